// Plan and launch of the few-row attention over a 4-bit cache (kernels: ma_decode.cuh).
#include "ma_kernels.cuh"

namespace ma {

int launch_decode_d64(const DecodeParams& p, int rows, bool wide, bool fast, cudaStream_t st);
int launch_decode_d128(const DecodeParams& p, int rows, bool wide, bool fast, cudaStream_t st);

namespace {

// Tiles that are contiguous in storage: positions packed back to back, K and V arrays of one
// geometry, 32-slot tiles that do not straddle pages, scale blocks on 16-byte boundaries.
bool contiguous_tiles(const ma_kv& kv, int D) {
  if (kv.mask != nullptr) return false;
  if (kv.pages != nullptr && kv.page_size % kDecodeTile != 0) return false;
  if (kv.skq[2] != D / 2 || kv.sks[2] != D / 32) return false;
  for (int i = 0; i < 3; ++i)
    if (kv.skq[i] != kv.svq[i] || kv.sks[i] != kv.svs[i] || (i < 2 && kv.sks[i] % 8 != 0)) return false;
  const uintptr_t bits = reinterpret_cast<uintptr_t>(kv.ks) | reinterpret_cast<uintptr_t>(kv.kz) |
                         reinterpret_cast<uintptr_t>(kv.vs) | reinterpret_cast<uintptr_t>(kv.vz);
  return (bits & 15) == 0;
}

// Rows per tile: a tile of more rows unpacks the codes fewer times, but 24 and 32 rows leave
// registers for 8 warps an SM only. 32 requests x 8192 slots, 4 KV heads, D = 128 (D = 64), us:
//   14 rows: 16 -> 59 (39), 24 -> 76 (50), 32 -> 98 (57)
//   21 rows: 16 -> 99 (67), 24 -> 81 (54), 32 -> 104 (61)
//   28 rows: 16 -> 100 (68), 24 -> 133 (88), 32 -> 107 (62)
//   35 rows: 16 -> 150 (93), 24 -> 135 (90), 32 -> 181 (103)
//   56 rows: 16 -> 194 (127), 24 -> 208 (140), 32 -> 184 (106)
// The general form has no 24-row tile.
int rows_per_tile(int R, int D, bool has24) {
  if (R <= 8) return 8;
  if (R <= 16) return 16;
  if (R <= 24) return has24 ? 24 : 32;
  if (R <= 32) return D == 64 ? 32 : 16;
  if (R <= 48) return has24 ? 24 : 16;
  return 32;
}

}  // namespace

void plan_decode(int B, int H, int R, int D, const ma_kv* kv, DecodePlan& plan) {
  const int sms = device_sm_count();
  plan.fast = kv == nullptr || contiguous_tiles(*kv, D);
  plan.wide = false;
  plan.rows = rows_per_tile(R, D, plan.fast);
  plan.row_tiles = (R + plan.rows - 1) / plan.rows;
  if (kv != nullptr) {
    // The wide form for few sequences and few units of slots by the cache's capacity (the lengths are on the
    // device), with the smallest tile of 8 or 16 rows that keeps to that: a tile's rows, not its slots, are
    // what a short call waits for. D = 128, us, wide 8 / 16 / 32 rows and the other form: 4 requests of up to 3227
    // slots, 2 heads, 64 rows 14 / 16 / 26 and 36; 1 x 8192, 4 heads, 21 rows 12 / 16 / 23 and 28; 1 x 39, 56 rows
    // 8 / 11 / 18 and 21; 16 of up to 3000, 2 heads, 32 rows (10 units an SM at 8 rows) 24 / 18. Beyond 8 units an SM
    // three 16-row tiles are still faster so (4 x 8192, 35 rows: 27 against 35; 56 rows: 38 against 49), one
    // or two are not (10 x 8192, 14 rows: 30 against 25; 8 x 8192, 21 rows: 36 against 35). More sequence heads
    // than SMs: 64 x 1000, 14 rows, 32 against 22.
    for (int rows = 8; rows <= 16 && !plan.wide; rows *= 2) {
      const int tiles = (R + rows - 1) / rows, most = rows == 16 && tiles >= 3 ? 16 : 8;
      const int64_t heads = (int64_t)B * H * tiles, units = heads * ((kv->nq + kDecodeUnit - 1) / kDecodeUnit);
      if (heads > sms || units > (int64_t)most * sms) continue;
      plan.wide = true;
      plan.rows = rows;
      plan.row_tiles = tiles;
    }
  }
  const bool three = plan.fast && (plan.rows == 8 || (plan.rows == 16 && D == 64));       // CTAs an SM, as launch_decode_d has them
  const int per_head = H * plan.row_tiles, resident = sms * (plan.wide ? 1 : three ? 3 : 2);
  plan.ctas = resident > per_head ? resident / per_head : 1;
}

// Bytes of partials for whichever form a call takes: at most 3 CTAs an SM, two partials each.
size_t decode_partials(int H, int R, int D, size_t& ml) {
  size_t most = 0;
  for (int rows = 8; rows <= 32; rows += 8) {
    const size_t tiles = (R + rows - 1) / rows, heads = (size_t)H * tiles;
    size_t ctas = (size_t)device_sm_count() * 3 / heads;
    if (ctas < 1) ctas = 1;
    const size_t splits = heads * 2 * ctas * rows;
    most = splits > most ? splits : most;
  }
  ml = (most * sizeof(float2) + 255) & ~(size_t)255;
  return ml + most * D * sizeof(float);
}

int launch_decode_attention(DecodeParams& p, const DecodePlan& plan, cudaStream_t st) {
  p.ctas = plan.ctas;
  p.row_tiles = plan.row_tiles;
  p.tiles_per_page = p.kv.pages != nullptr ? p.kv.page_size / kDecodeTile : 1;
  p.kchan_vec = ((reinterpret_cast<uintptr_t>(p.kv.kchan) & 15) == 0 && p.kv.skc[0] % 4 == 0 && p.kv.skc[1] % 4 == 0) ? 1 : 0;
  p.tile_div.set(p.tiles_per_page > 0 ? p.tiles_per_page : 1);
  return p.D == 128 ? launch_decode_d128(p, plan.rows, plan.wide, plan.fast, st)
                    : launch_decode_d64(p, plan.rows, plan.wide, plan.fast, st);
}

}  // namespace ma
