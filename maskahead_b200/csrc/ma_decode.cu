// Attention of few query rows (single tokens, short drafts) over a token-mode k4v4 cache read
// in place, contiguous or paged, and over the step's own bf16 keys (token-causal).
//
// For row r of KV head h, slot j with codes c, scale s_g and zero z_g per 32-channel group:
//     score = scale * sum_d q_d kchan_d (c_d s_g + z_g)
//           = scale * sum_g ( s_g * sum_{d in g} q'_d c_d  +  z_g * sum_{d in g} q'_d ),  q' = q kchan
//     out   = sum_j p_j (c_d s_g + z_g) = sum_j (p_j s_g) c_d + sum_j p_j z_g
// so the codes enter the matrix products as they are and only per-slot factors touch fp32: no
// element is ever dequantized. A code of 4 bits masked out of its byte IS an fp16 subnormal,
// c * 2^-24 (or c * 2^-20 from the high nibble), exact for the fp16 MMA; one shift and four
// masks turn a 32-bit word into the A operands of eight codes.
//
// Bound: HBM (160 B per slot and KV head at D = 128) while the rows fit one or two 8-column
// MMA tiles, the issue slots beyond. The rows are the N side (8 columns) of m16n8k16, the slots
// (scores) or channels (output) its M side: G = 7 single-token rows waste one column of eight,
// where a 128-row tcgen05 tile would waste 121 of 128 and need the codes written back to
// shared memory as 16-bit operands first, 3.2 times their stored size.
//
// A warp owns 32-slot tiles and a private ring of shared memory filled by cp.async (16-byte
// payload pieces in an XOR swizzle that ldmatrix reads without conflicts, 8-byte scale and
// zero rows), so the main loop has no CTA barrier. Splits: every CTA derives the chunk length
// from the lengths on the device (they are not known on the host), writes fp32 partials,
// and the last CTA of a (sequence, head, row tile) merges them; nobody waits.
#include "ma_kernels.cuh"

namespace ma {

namespace {

constexpr int kTile = 32;                 // slots per warp tile
constexpr int kUnit = 256;                // chunk granularity in slots
constexpr int kStages = 2;
constexpr float kLog2e = 1.4426950408889634f;

// Shared memory of one ring stage: K payload, V payload (D/2 bytes a slot each), then the
// K scale, K zero, V scale and V zero rows (D/16 bytes a slot each).
template <int D>
struct Ring {
  static constexpr int kPay = kTile * (D / 2);
  static constexpr int kSc = kTile * (D / 16);
  static constexpr int kVq = kPay, kKs = 2 * kPay, kKz = kKs + kSc, kVs = kKz + kSc, kVz = kVs + kSc;
  static constexpr int kStage = kVz + kSc;
  static constexpr int kWarpBytes = kStages * kStage;
  static_assert(kStage % 128 == 0, "stages keep the swizzle's 128-byte phase");
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
template <int N>
__device__ __forceinline__ void cp_async(uint32_t dst, const void* src, uint32_t bytes) {
  // bytes = N, or 0: the destination is zero-filled and the source not read
  if constexpr (N == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;\n" ::"r"(dst), "l"(src), "n"(N), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldsm4(uint32_t r[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t r[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void mma16(float c[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                      uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma8(float c[4], uint32_t a0, uint32_t a1, uint32_t b0) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%7,%7,%7,%7};\n"
               : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(b0), "f"(0.f));
}
// the first product of a sum: c = a b
__device__ __forceinline__ void mma16_set(float c[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
               : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];\n" : "=r"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t lds16(uint32_t a) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];\n" : "=h"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];\n" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  __half2 r = __hmul2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<uint32_t*>(&r);
}
__device__ __forceinline__ float2 half2_floats(uint32_t a) { return __half22float2(*reinterpret_cast<__half2*>(&a)); }

// 16-byte piece c of slot s's payload row within a stage's payload block
template <int D>
__device__ __forceinline__ uint32_t piece(int s, int c) {
  if constexpr (D == 128) return s * 64 + ((c ^ ((s >> 1) & 3)) << 4);
  return s * 32 + ((c ^ ((s >> 2) & 1)) << 4);
}

// Where CTA x works.
struct Split {
  int b;          // sequence, -1: nothing to do
  int chunk;      // chunk of its prefix, or -1: the block's own keys
  int per;        // chunk length in units of kUnit slots
  int first;      // partial slot of its first chunk
  int count;      // partials of this sequence (chunks, plus the block)
  int total;      // chunks of every sequence
};

__device__ __forceinline__ int live_slots(const DecodeParams& p, int b) {
  int n = p.kv.nq;
  if (p.kv.lens != nullptr) n = min(n, max(p.kv.lens[b], 0));
  return n;
}

// The work of CTA x: the chunk length that spreads every sequence's live slots over about
// `target` CTAs, then the CTA's place in the list of chunks (each warp computes it alone).
__device__ __forceinline__ Split find_split(const DecodeParams& p, int x, int lane) {
  const int least = p.cur.Tc > 0 ? 0 : 1;      // a sequence without any key still writes its rows
  int units = 0;
  for (int b = lane; b < p.B; b += 32) units += (live_slots(p, b) + kUnit - 1) / kUnit;
  units = __reduce_add_sync(0xffffffffu, units);
  Split s;
  s.per = max(p.min_units, (units + p.target - 1) / p.target);
  s.b = -1;
  s.chunk = -1;
  int at = 0;
  for (int b0 = 0; b0 < p.B; b0 += 32) {
    const int b = b0 + lane;
    int n = 0;
    if (b < p.B) n = max(least, ((live_slots(p, b) + kUnit - 1) / kUnit + s.per - 1) / s.per);
    int incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    const int excl = at + incl - n;
    const unsigned hit = __ballot_sync(0xffffffffu, b < p.B && x >= excl && x < at + incl);
    if (hit) {
      const int src = __ffs(hit) - 1;
      s.b = b0 + src;
      s.first = __shfl_sync(0xffffffffu, excl, src);
      s.count = __shfl_sync(0xffffffffu, n, src);
      s.chunk = x - s.first;
    }
    at += __shfl_sync(0xffffffffu, incl, 31);
  }
  s.total = at;
  if (p.cur.Tc > 0) {
    if (s.b < 0 && x - at < p.B) {      // the block's keys of sequence x - at
      s.b = x - at;
      const int units_b = (live_slots(p, s.b) + kUnit - 1) / kUnit;
      s.count = (units_b + s.per - 1) / s.per;
      // its chunks' place: counted again up to this sequence
      int before = 0;
      for (int b = lane; b < s.b; b += 32) before += ((live_slots(p, b) + kUnit - 1) / kUnit + s.per - 1) / s.per;
      s.first = __reduce_add_sync(0xffffffffu, before);
    }
    s.count += 1;
  }
  return s;
}

template <int D>
__device__ __forceinline__ void store_row4(const DecodeParams& p, int b, int h, int r, int d, float4 o) {
  const int g = r / p.T, t = r - g * p.T;
  __nv_bfloat16* dst = p.out + (int64_t)b * p.so[0] + (int64_t)(h * p.G + g) * p.so[1] + (int64_t)t * p.so[2] + d;
  store4(dst, o.x, o.y, o.z, o.w);
}

// A CTA's result from nsrc sources in shared memory -- sRows[nsrc][ROWS][kPad] unnormalized
// rows, sML[nsrc][ROWS] their (m, l) -- to the output rows (normalized) or to partial `slot`.
template <int D, int ROWS, int W>
__device__ __forceinline__ void combine(const DecodeParams& p, int b, int h, int r0, int rows, int nsrc, const float* sRows,
                                        const float2* sML, float2* ml, float* acc) {
  constexpr int kVec = D / 4, kPad = D + 4;
  for (int i = threadIdx.x; i < rows * kVec; i += W * 32) {
    const int r = i / kVec, d = (i % kVec) * 4;
    float m = -INFINITY;
    for (int w = 0; w < nsrc; ++w) m = fmaxf(m, sML[w * ROWS + r].x);
    const float ms = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int w = 0; w < nsrc; ++w) {
      const float2 e = sML[w * ROWS + r];
      const float f = ex2(e.x - ms);
      const float4 v = *reinterpret_cast<const float4*>(sRows + (w * ROWS + r) * kPad + d);
      l = fmaf(f, e.y, l);
      o.x = fmaf(f, v.x, o.x);
      o.y = fmaf(f, v.y, o.y);
      o.z = fmaf(f, v.z, o.z);
      o.w = fmaf(f, v.w, o.w);
    }
    if (acc == nullptr) {
      const float inv = l > 0.f ? 1.f / l : 0.f;
      store_row4<D>(p, b, h, r0 + r, d, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
    } else {
      __stcg(reinterpret_cast<float4*>(acc + r * D + d), o);
      if (d == 0) __stcg(&ml[r], make_float2(m, l));
    }
  }
}

// The merge of a sequence's partials, in the last of its CTAs: warp w folds splits w, w + W, ...
// into running rows (8 rows at a time, two splits in flight), then the warps' rows are combined
// as a CTA's own are. The order is fixed, so the result does not depend on who came last.
template <int D, int ROWS, int W>
__device__ void merge_partials(const DecodeParams& p, const Split& s, int b, int h, int r0, int rows, const float2* ml,
                               const float* acc, float* sRows, float2* sML) {
  constexpr int kPad = D + 4, kLanes = D / 4;         // lanes of a row; with 64 channels a warp reads two at once
  constexpr int kPer = 32 / kLanes, kStep = 8 / kPer;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int chunks = p.cur.Tc > 0 ? s.count - 1 : s.count;
  const int sub = lane / kLanes, d = (lane % kLanes) * 4;
  for (int g0 = 0; g0 < rows; g0 += 8) {
    float m = -INFINITY, l = 0.f;                     // of row g0 + lane (lanes 0 .. 7)
    float4 o[kStep];
#pragma unroll
    for (int k = 0; k < kStep; ++k) o[k] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i = warp; i < s.count; i += 2 * W) {
      float2 e[2];
      float4 v[2][kStep];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int x = i + u * W;
        e[u] = make_float2(-INFINITY, 0.f);
        if (x < s.count) {
          const int64_t at = (int64_t)(x < chunks ? s.first + x : s.total + b) * ROWS + g0;
          if (lane < 8 && g0 + lane < rows) e[u] = __ldcg(&ml[at + lane]);
#pragma unroll
          for (int k = 0; k < kStep; ++k) {
            const int r = k * kPer + sub;
            v[u][k] = g0 + r < rows ? __ldcg(reinterpret_cast<const float4*>(acc + (at + r) * D + d))
                                    : make_float4(0.f, 0.f, 0.f, 0.f);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (i + u * W >= s.count) break;
        const float mn = fmaxf(m, e[u].x), ms = mn == -INFINITY ? 0.f : mn;
        const float old = ex2(m - ms), add = ex2(e[u].x - ms);
        m = mn;
        l = l * old + e[u].y * add;
#pragma unroll
        for (int k = 0; k < kStep; ++k) {
          const float f = __shfl_sync(0xffffffffu, old, k * kPer + sub), w = __shfl_sync(0xffffffffu, add, k * kPer + sub);
          o[k].x = fmaf(w, v[u][k].x, o[k].x * f);
          o[k].y = fmaf(w, v[u][k].y, o[k].y * f);
          o[k].z = fmaf(w, v[u][k].z, o[k].z * f);
          o[k].w = fmaf(w, v[u][k].w, o[k].w * f);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < kStep; ++k)
      *reinterpret_cast<float4*>(sRows + (warp * ROWS + g0 + k * kPer + sub) * kPad + d) = o[k];
    if (lane < 8) sML[warp * ROWS + g0 + lane] = make_float2(m, l);
  }
  __syncthreads();
  combine<D, ROWS, W>(p, b, h, r0, rows, W, sRows, sML, nullptr, nullptr);
}

// The CTA's rows: the output when they are the sequence's only split, else this split's partial
// and, in the last CTA to arrive, the merge of all of them.
template <int D, int ROWS, int W>
__device__ void finish(const DecodeParams& p, const Split& s, int h, int rt, int slot, int nsrc, float* sRows, float2* sML,
                       float2* sMerge) {
  __shared__ int sLast;
  const int r0 = rt * ROWS, rows = min(ROWS, p.R - r0);
  const int b = s.b;
  if (s.count == 1) {
    combine<D, ROWS, W>(p, b, h, r0, rows, nsrc, sRows, sML, nullptr, nullptr);
    return;
  }
  const int64_t base = (int64_t)(h * p.row_tiles + rt) * p.slots * ROWS;
  float2* ml = p.ml + base;
  float* acc = p.acc + base * D;
  combine<D, ROWS, W>(p, b, h, r0, rows, nsrc, sRows, sML, ml + (int64_t)slot * ROWS, acc + (int64_t)slot * ROWS * D);
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    unsigned* ticket = p.tickets + ((int64_t)b * p.H + h) * p.row_tiles + rt;
    const unsigned got = atomicAdd(ticket, 1u);
    sLast = got == (unsigned)s.count - 1u;
    if (sLast) *ticket = 0u;      // ready for the next call
  }
  __syncthreads();
  if (!sLast) return;
  __threadfence();
  merge_partials<D, ROWS, W>(p, s, b, h, r0, rows, ml, acc, sRows, sMerge);
}

// The step's own keys: a warp per row, a lane per key, in fp32 (a few hundred products a row).
template <int D, int ROWS, int W>
__device__ void block_split(const DecodeParams& p, const Split& s, int h, int rt, char* smem) {
  constexpr int kPad = D + 4;
  constexpr int kRow = D + 8;                              // staged bf16 row, 16 bytes of padding
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = s.b, r0 = rt * ROWS, rows = min(ROWS, p.R - r0);
  float2* sML = reinterpret_cast<float2*>(smem);            // [W][ROWS]
  float* sRows = reinterpret_cast<float*>(smem + W * ROWS * 8);     // [W][ROWS][kPad]: q first, the result later
  __nv_bfloat16* sK = reinterpret_cast<__nv_bfloat16*>(smem + W * ROWS * 8 + ROWS * kPad * 4);
  __nv_bfloat16* sV = sK + 32 * kRow;
  const __nv_bfloat16* K = reinterpret_cast<const __nv_bfloat16*>(p.cur.k) + (int64_t)b * p.cur.sk[0] + (int64_t)h * p.cur.sk[1];
  const __nv_bfloat16* V = reinterpret_cast<const __nv_bfloat16*>(p.cur.v) + (int64_t)b * p.cur.sv[0] + (int64_t)h * p.cur.sv[1];
  for (int i = tid; i < rows * (D / 8); i += W * 32) {
    const int r = i / (D / 8), d = (i % (D / 8)) * 8;
    const int g = (r0 + r) / p.T, t = (r0 + r) - g * p.T;
    float f[8];
    load8(p.q + (int64_t)b * p.sq[0] + (int64_t)(h * p.G + g) * p.sq[1] + (int64_t)t * p.sq[2] + d, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) sRows[r * kPad + d + e] = f[e];
  }
  constexpr int kOwn = (ROWS + W - 1) / W;                       // rows per warp
  constexpr int kCh = D / 32;                               // channels per lane
  float m[kOwn], l[kOwn], o[kOwn][kCh];
#pragma unroll
  for (int i = 0; i < kOwn; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int c = 0; c < kCh; ++c) o[i][c] = 0.f;
  }
  for (int j0 = 0; j0 < p.cur.Tc; j0 += 32) {
    const int nj = min(32, p.cur.Tc - j0);
    __syncthreads();
    for (int i = tid; i < 32 * (D / 8); i += W * 32) {
      const int j = i / (D / 8), d = (i % (D / 8)) * 8;
      uint4 kv = make_uint4(0u, 0u, 0u, 0u), vv = kv;
      if (j < nj) {
        kv = *reinterpret_cast<const uint4*>(K + (int64_t)(j0 + j) * p.cur.sk[2] + d);
        vv = *reinterpret_cast<const uint4*>(V + (int64_t)(j0 + j) * p.cur.sv[2] + d);
      }
      *reinterpret_cast<uint4*>(sK + j * kRow + d) = kv;
      *reinterpret_cast<uint4*>(sV + j * kRow + d) = vv;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      const int r = warp + i * W;
      if (r >= rows) break;
      const int t = (r0 + r) % p.T;
      const int seen = p.causal ? t + p.cur.Tc - p.T : p.cur.Tc - 1;    // the last key this row sees
      float dot = 0.f;
#pragma unroll 4
      for (int d = 0; d < D; d += 8) {
        float kf[8];
        bf16x8_to_float(*reinterpret_cast<const uint4*>(sK + lane * kRow + d), kf);
        const float4 qa = *reinterpret_cast<const float4*>(sRows + r * kPad + d);
        const float4 qb = *reinterpret_cast<const float4*>(sRows + r * kPad + d + 4);
        dot = fmaf(qa.x, kf[0], dot); dot = fmaf(qa.y, kf[1], dot); dot = fmaf(qa.z, kf[2], dot);
        dot = fmaf(qa.w, kf[3], dot); dot = fmaf(qb.x, kf[4], dot); dot = fmaf(qb.y, kf[5], dot);
        dot = fmaf(qb.z, kf[6], dot); dot = fmaf(qb.w, kf[7], dot);
      }
      const float sc = (lane < nj && j0 + lane <= seen) ? dot * p.scale * kLog2e : -INFINITY;
      const float mn = fmaxf(m[i], warp_max(sc));
      const float ms = mn == -INFINITY ? 0.f : mn;
      const float corr = ex2(m[i] - ms), pr = ex2(sc - ms);
      m[i] = mn;
      l[i] = l[i] * corr + warp_sum(pr);
#pragma unroll
      for (int c = 0; c < kCh; ++c) o[i][c] *= corr;
      for (int j = 0; j < nj; ++j) {
        const float w = __shfl_sync(0xffffffffu, pr, j);
        if (w == 0.f) continue;              // a key this row does not see: its value is not read
#pragma unroll
        for (int c = 0; c < kCh; ++c) o[i][c] = fmaf(w, __bfloat162float(sV[j * kRow + lane * kCh + c]), o[i][c]);
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kOwn; ++i) {
    const int r = warp + i * W;
    if (r >= rows) break;
#pragma unroll
    for (int c = 0; c < kCh; ++c) sRows[r * kPad + lane * kCh + c] = o[i][c];
    if (lane == 0) sML[r] = make_float2(m[i], l[i]);
  }
  __syncthreads();
  finish<D, ROWS, W>(p, s, h, rt, s.total + b, 1, sRows, sML, sML);
}

// FAST: tiles are contiguous in storage (launch() says when); else every slot is looked up alone.
template <int D, int NT, int W, int MINB, bool FAST>
__global__ void __launch_bounds__(W * 32, MINB) decode_attention_kernel(const __grid_constant__ DecodeParams p) {
  constexpr int ROWS = 8 * NT, NG = D / 32, kPad = D + 4, kSc = D / 16;
  using R = Ring<D>;
  extern __shared__ __align__(128) char smem[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t4 = lane & 3;
  const int h = blockIdx.y / p.row_tiles, rt = blockIdx.y - h * p.row_tiles;
  const Split s = find_split(p, blockIdx.x, lane);
  if (s.b < 0) return;
  const int b = s.b;
  if (s.chunk < 0) {
    block_split<D, ROWS, W>(p, s, h, rt, smem);
    return;
  }
  const ma_kv& kv = p.kv;
  const int n = live_slots(p, b);
  const int64_t begin = (int64_t)s.chunk * s.per * kUnit;
  const int end = (int)min((int64_t)n, begin + (int64_t)s.per * kUnit);
  const uint32_t ring = smem_u32(smem) + warp * R::kWarpBytes;

  // ---- the copies of a tile of 32 slots into a ring stage. `find` looks a tile up (a load from
  // the page table, one tile ahead of its use), `issue` starts its copies and returns its live
  // slots; dead ones are zero-filled, so nothing stored there is ever multiplied.
  const int tiles = end > begin ? (int)((end - begin + kTile - 1) / kTile) : 0;
  constexpr int kPieces = D / 32, kSlots = 32 / kPieces;       // 16-byte pieces per slot, slots per pass
  struct Place {
    int page, at;      // FAST: of the tile, else of this lane's slot; page -1: dead
  };
  const int64_t hq = (int64_t)h * kv.skq[1], hs = (int64_t)h * kv.sks[1], hvq = (int64_t)h * kv.svq[1], hvs = (int64_t)h * kv.svs[1];
  auto find = [&](int i) -> Place {
    Place f = {-1, 0};
    if constexpr (FAST) {
      if (i < tiles) {
        const int x = (int)(begin / kTile) + i;
        f.page = b;
        f.at = x;
        if (kv.pages != nullptr) {
          const int pi = p.tile_div.div(x);
          f.at = x - pi * p.tiles_per_page;
          f.page = kv.pages[(int64_t)b * kv.spg + pi];
          if ((unsigned)f.page >= (unsigned)kv.num_pages) f.page = -1;
        }
      }
    } else {
      const int64_t j = begin + (int64_t)i * kTile + lane;
      if (i < tiles && j < end) {
        kv_page(kv, b, (int)j, f.page, f.at);
        if (kv.mask != nullptr && kv.mask[((int64_t)b * p.H + h) * kv.nq + j] == 0) f.page = -1;
      }
    }
    return f;
  };
  // FAST: this lane's share of a tile's contiguous 32 D/2 payload bytes and, in the order they
  // have in a stage, of the four scale and zero blocks
  constexpr int kScPieces = kTile * kSc / 16, kScLanes = kTile / kScPieces;    // 16-byte pieces per block, slots each
  const char* lane_sc[NG / 2];
#pragma unroll
  for (int it = 0; it < NG / 2; ++it) {
    const int blk = (it * 32 + lane) / kScPieces;
    const uint16_t* base = blk == 0 ? kv.ks + hs : blk == 1 ? kv.kz + hs : blk == 2 ? kv.vs + hvs : kv.vz + hvs;
    lane_sc[it] = reinterpret_cast<const char*>(base) + (lane % kScPieces) * 16;
  }
  const uint8_t* lane_kq = kv.kq + hq + (FAST ? lane * 16 : 0);
  const uint8_t* lane_vq = kv.vq + hvq + (FAST ? lane * 16 : 0);
  auto issue = [&](int i, int stage, Place f) -> unsigned {
    unsigned alive;
    const uint32_t st = ring + stage * R::kStage;
    if constexpr (FAST) {
      const int64_t left = end - (begin + (int64_t)i * kTile);
      const int cnt = f.page < 0 ? 0 : (int)min((int64_t)kTile, left);
      alive = cnt == kTile ? 0xffffffffu : (1u << cnt) - 1u;
      if (i < tiles) {
        const int64_t pg = max(f.page, 0);
        const int64_t oq = pg * kv.skq[0] + (int64_t)f.at * (kTile * D / 2), os = (pg * kv.sks[0] + (int64_t)f.at * (kTile * NG)) * 2;
#pragma unroll
        for (int it = 0; it < kPieces; ++it) {
          const int sl = it * kSlots + lane / kPieces, c = lane % kPieces;
          const uint32_t bytes = sl < cnt ? 16u : 0u;
          cp_async<16>(st + piece<D>(sl, c), lane_kq + oq + it * 512, bytes);
          cp_async<16>(st + R::kVq + piece<D>(sl, c), lane_vq + oq + it * 512, bytes);
        }
        const int sc_left = (cnt - (lane % kScPieces) * kScLanes) * kSc;
        const uint32_t bytes = min(max(sc_left, 0), 16);
#pragma unroll
        for (int it = 0; it < NG / 2; ++it) cp_async<16>(st + R::kKs + (it * 32 + lane) * 16, lane_sc[it] + os, bytes);
      }
    } else {
      const bool live = f.page >= 0;
      alive = __ballot_sync(0xffffffffu, live);
      if (i < tiles) {
        const int64_t pb = live ? f.page : 0, pj = live ? f.at : 0;
        const int64_t okq = pb * kv.skq[0] + pj * kv.skq[2], ovq = pb * kv.svq[0] + pj * kv.svq[2];
        const int64_t oks = hs + pb * kv.sks[0] + pj * kv.sks[2], ovs = hvs + pb * kv.svs[0] + pj * kv.svs[2];
        const uint32_t sc = live ? kSc : 0;
        cp_async<kSc>(st + R::kKs + lane * kSc, kv.ks + oks, sc);
        cp_async<kSc>(st + R::kKz + lane * kSc, kv.kz + oks, sc);
        cp_async<kSc>(st + R::kVs + lane * kSc, kv.vs + ovs, sc);
        cp_async<kSc>(st + R::kVz + lane * kSc, kv.vz + ovs, sc);
#pragma unroll
        for (int it = 0; it < kPieces; ++it) {
          const int sl = it * kSlots + lane / kPieces, c = lane % kPieces;
          const int64_t ok = __shfl_sync(0xffffffffu, okq, sl), ov = __shfl_sync(0xffffffffu, ovq, sl);
          const uint32_t bytes = (alive >> sl & 1u) ? 16u : 0u;
          cp_async<16>(st + piece<D>(sl, c), lane_kq + ok + c * 16, bytes);
          cp_async<16>(st + R::kVq + piece<D>(sl, c), lane_vq + ov + c * 16, bytes);
        }
      }
    }
    cp_commit();
    return alive;
  };

  unsigned flight[kStages];        // live slots of the tiles in flight, the next tile's first
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) flight[i] = issue(warp + i * W, i, find(warp + i * W));
  Place next = find(warp + (kStages - 1) * W);

  // ---- the query rows as B operands: q' = q kchan in fp16, scaled by a power of two so that a
  // row's largest magnitude lies in [2^13, 2^14) (11 bits of q', where a bf16 cache would
  // round k to 8). Thread (g, t4) holds channels 32 gr + 8 t4 + 0..7 of row g; the products pair
  // channels (0, 4), (1, 5), (2, 6), (3, 7) of a word as its masks leave them, the odd ones with
  // q' / 16 because a high nibble is worth 16 times a low one.
  uint32_t qb[NT][NG][4], zb[NT];
  float fr[NT][2];                 // score in log2 units = fr * sum, fr > 0: the scale's sign goes into q'
  const float sign = p.scale > 0.f ? 1.f : p.scale < 0.f ? -1.f : 0.f, size = p.scale == 0.f ? 1.f : fabsf(p.scale);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = rt * ROWS + nt * 8 + g;
    float x[NG][8], amax = 0.f;
    const int rg = r / p.T, rt_ = r - rg * p.T;
    const __nv_bfloat16* q = p.q + (int64_t)b * p.sq[0] + (int64_t)(h * p.G + rg) * p.sq[1] + (int64_t)rt_ * p.sq[2];
    const float* kc = kv.kchan + (int64_t)b * kv.skc[0] + (int64_t)h * kv.skc[1];
#pragma unroll
    for (int gr = 0; gr < NG; ++gr) {
      const int d = 32 * gr + 8 * t4;
      if (r < p.R) {
        load8(q + d, x[gr]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[gr][e] = 0.f;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[gr][e] *= kc[d + e] * sign;
        amax = fmaxf(amax, fabsf(x[gr][e]));
      }
    }
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    const int eb = min(max((int)(__float_as_uint(amax) >> 23), 16), 240);
    const float up = __uint_as_float((uint32_t)(267 - eb) << 23);       // 2^(13 - exponent)
    float zg[NG];
#pragma unroll
    for (int gr = 0; gr < NG; ++gr) {
      float z = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[gr][e] = __half2float(__float2half_rn(x[gr][e] * up));
        z += x[gr][e];
      }
      qb[nt][gr][0] = pack_half2(x[gr][0], x[gr][4]);
      qb[nt][gr][1] = pack_half2(x[gr][1] * 0.0625f, x[gr][5] * 0.0625f);
      qb[nt][gr][2] = pack_half2(x[gr][2], x[gr][6]);
      qb[nt][gr][3] = pack_half2(x[gr][3] * 0.0625f, x[gr][7] * 0.0625f);
      z += __shfl_xor_sync(0xffffffffu, z, 1);
      z += __shfl_xor_sync(0xffffffffu, z, 2);
      zg[gr] = z * 5.9604645e-8f;  // 2^-24, the unit of the codes' products
    }
    // the groups' sums of q' for the zero term, as fp16 high and low parts: together exact to
    // half a unit of q', below q's own rounding
    float z0, z1;
    bool low;
    if constexpr (NG == 4) {
      z0 = (t4 & 1) ? zg[2] : zg[0];
      z1 = (t4 & 1) ? zg[3] : zg[1];
      low = t4 >= 2;
    } else {
      z0 = t4 < 2 ? zg[0] : 0.f;
      z1 = t4 < 2 ? zg[1] : 0.f;
      low = t4 & 1;
    }
    const float h0 = __half2float(__float2half_rn(z0)), h1 = __half2float(__float2half_rn(z1));
    zb[nt] = low ? pack_half2(z0 - h0, z1 - h1) : pack_half2(h0, h1);
    const float f = size * kLog2e * 16777216.f * __uint_as_float((uint32_t)(eb - 13) << 23);
    fr[nt][0] = __shfl_sync(0xffffffffu, f, 8 * t4);        // rows 2 t4 and 2 t4 + 1: the lanes that hold them as g
    fr[nt][1] = __shfl_sync(0xffffffffu, f, 8 * t4 + 4);
  }

  float o[NT][NG][8], zl[NT][2], m[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    zl[nt][0] = zl[nt][1] = 0.f;
    m[nt][0] = m[nt][1] = -INFINITY;
#pragma unroll
    for (int gr = 0; gr < NG; ++gr)
#pragma unroll
      for (int i = 0; i < 8; ++i) o[nt][gr][i] = 0.f;
  }
  int fe = 14;                     // the V scales are multiplied by 2^fe so that the largest lies below 2

  // the zero term's A rows: 0 .. NG-1 the groups' zeros, 4 ones, the others nothing
  const uint32_t zkeep = g < NG ? 0xffffffffu : 0u, zone = g == 4 ? 0x3C003C00u : 0u;
  // ldmatrix rows of this lane: matrix mi = lane / 8 covers slots 8 (mi & 1) .. + 7 of group mi / 2
  const int lm_slot = (lane & 7) + ((lane >> 3) & 1) * 8, lm_grp = lane >> 4;

  int stage = 0;                   // ring stage of tile i; tile i + kStages - 1 goes into the one before it
  for (int i = warp; i < tiles; i += W) {
    const int nx = i + (kStages - 1) * W;
    flight[kStages - 1] = issue(nx, stage == 0 ? kStages - 1 : stage - 1, next);
    next = find(nx + W);
    cp_wait<kStages - 1>();
    __syncwarp();
    const uint32_t st = ring + stage * R::kStage;
    const unsigned alive = flight[0];
#pragma unroll
    for (int e = 0; e < kStages - 1; ++e) flight[e] = flight[e + 1];
    stage = stage == kStages - 1 ? 0 : stage + 1;

    // ---- scores of 2 x 16 slots
    float sc[2][NT][4];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      const uint32_t sa = st + (mt * 16 + g) * kSc;
      float s0[NG], s1[NG];
      if constexpr (NG == 4) {
        const uint2 u0 = lds64(sa + R::kKs), u1 = lds64(sa + R::kKs + 8 * kSc);
        const float2 a = half2_floats(u0.x), c = half2_floats(u0.y), e = half2_floats(u1.x), f = half2_floats(u1.y);
        s0[0] = a.x; s0[1] = a.y; s0[2] = c.x; s0[3] = c.y;
        s1[0] = e.x; s1[1] = e.y; s1[2] = f.x; s1[3] = f.y;
      } else {
        const float2 a = half2_floats(lds32(sa + R::kKs)), c = half2_floats(lds32(sa + R::kKs + 8 * kSc));
        s0[0] = a.x; s0[1] = a.y; s1[0] = c.x; s1[1] = c.y;
      }
      const uint32_t za = sa + R::kKz + (NG == 4 ? (t4 & 1) * 4 : 0);
      const uint32_t z0 = lds32(za), z1 = lds32(za + 8 * kSc);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) mma8(sc[mt][nt], z0, z1, zb[nt]);
#pragma unroll
      for (int gp = 0; gp < NG / 2; ++gp) {
        uint32_t w[4];
        ldsm4(w, st + piece<D>(mt * 16 + lm_slot, gp * 2 + lm_grp));
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int gr = gp * 2 + e;
          const uint32_t wa = w[2 * e], wb = w[2 * e + 1], xa = wa >> 8, xb = wb >> 8;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float c[4];
            mma16_set(c, wa & 0x000F000Fu, wb & 0x000F000Fu, wa & 0x00F000F0u, wb & 0x00F000F0u, qb[nt][gr][0], qb[nt][gr][1]);
            mma16(c, xa & 0x000F000Fu, xb & 0x000F000Fu, xa & 0x00F000F0u, xb & 0x00F000F0u, qb[nt][gr][2], qb[nt][gr][3]);
            sc[mt][nt][0] = fmaf(s0[gr], c[0], sc[mt][nt][0]);
            sc[mt][nt][1] = fmaf(s0[gr], c[1], sc[mt][nt][1]);
            sc[mt][nt][2] = fmaf(s1[gr], c[2], sc[mt][nt][2]);
            sc[mt][nt][3] = fmaf(s1[gr], c[3], sc[mt][nt][3]);
          }
        }
      }
    }
    if (alive != 0xffffffffu) {
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!(alive >> (mt * 16 + (e >> 1) * 8 + g) & 1u)) sc[mt][nt][e] = -INFINITY;
    }

    // ---- the tile's largest V scale, as an exponent
    uint32_t top;
    if constexpr (NG == 4) {
      const uint2 u = lds64(st + R::kVs + lane * kSc);
      const uint32_t a = __vmaxu2(u.x & 0x7fff7fffu, u.y & 0x7fff7fffu);
      top = max(a & 0xffffu, a >> 16);
    } else {
      const uint32_t a = lds32(st + R::kVs + lane * kSc) & 0x7fff7fffu;
      top = max(a & 0xffffu, a >> 16);
    }
    top = __reduce_max_sync(0xffffffffu, top);
    const int fe_new = min(fe, 15 - min(max((int)(top >> 10), 1), 30));
    const float down = __uint_as_float((uint32_t)(127 + fe_new - fe) << 23);
    fe = fe_new;
    const uint32_t fh = fe > -15 ? (uint32_t)(fe + 15) << 10 : 0x0200u;
    const uint32_t up2 = fh | fh << 16;

    // ---- softmax: running maximum per row over the tile's 32 slots; p in units of 2^-14 so that
    // fp16 keeps 11 bits of it down to 2^-28 of the row's maximum
    float corr[NT][2];
    uint32_t pb[2][NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float off[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float v = fmaxf(fmaxf(sc[0][nt][c], sc[0][nt][c + 2]), fmaxf(sc[1][nt][c], sc[1][nt][c + 2]));
        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
        const float mn = fmaxf(m[nt][c], v);
        const float ms = mn == -INFINITY ? 0.f : mn;
        corr[nt][c] = ex2((m[nt][c] - ms) * fr[nt][c]);
        m[nt][c] = mn;
        off[c] = fmaf(-ms, fr[nt][c], 14.f);
      }
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        pb[mt][nt][0] = transpose8x8(pack_half2(ex2(fmaf(sc[mt][nt][0], fr[nt][0], off[0])),
                                                 ex2(fmaf(sc[mt][nt][1], fr[nt][1], off[1]))));
        pb[mt][nt][1] = transpose8x8(pack_half2(ex2(fmaf(sc[mt][nt][2], fr[nt][0], off[0])),
                                                 ex2(fmaf(sc[mt][nt][3], fr[nt][1], off[1]))));
      }
    }

    // ---- zero term and row sum: A rows 0 .. NG-1 hold the slots' V zeros, row 4 ones
    {
      uint32_t a[2][2];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int hb = 0; hb < 2; ++hb) {
          const uint32_t za = st + R::kVz + (mt * 16 + hb * 8 + 2 * t4) * kSc + (g & (NG - 1)) * 2;
          a[mt][hb] = (__byte_perm(lds16(za), lds16(za + kSc), 0x5410) & zkeep) | zone;
        }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float c[4];
        mma16_set(c, a[0][0], 0u, a[0][1], 0u, pb[0][nt][0], pb[0][nt][1]);
        mma16(c, a[1][0], 0u, a[1][1], 0u, pb[1][nt][0], pb[1][nt][1]);
        zl[nt][0] = fmaf(zl[nt][0], corr[nt][0], c[0]);
        zl[nt][1] = fmaf(zl[nt][1], corr[nt][1], c[1]);
      }
    }

    // ---- V scales of the slots this lane's B operands hold, in pairs of slots
    uint32_t vsc[2][2][NG];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int hb = 0; hb < 2; ++hb) {
        const uint32_t va = st + R::kVs + (mt * 16 + hb * 8 + 2 * t4) * kSc;
        if constexpr (NG == 4) {
          const uint4 u = lds128(va);
          vsc[mt][hb][0] = hmul2(__byte_perm(u.x, u.z, 0x5410), up2);
          vsc[mt][hb][1] = hmul2(__byte_perm(u.x, u.z, 0x7632), up2);
          vsc[mt][hb][2] = hmul2(__byte_perm(u.y, u.w, 0x5410), up2);
          vsc[mt][hb][3] = hmul2(__byte_perm(u.y, u.w, 0x7632), up2);
        } else {
          const uint2 u = lds64(va);
          vsc[mt][hb][0] = hmul2(__byte_perm(u.x, u.y, 0x5410), up2);
          vsc[mt][hb][1] = hmul2(__byte_perm(u.x, u.y, 0x7632), up2);
        }
      }

    // ---- codes' part of the output. The tile's products are summed from zero and added to the
    // running sum in fp32: the codes are not centred, so a long chain of the tensor core's
    // truncating additions would leave a bias in the difference of the two parts.
#pragma unroll
    for (int gp = 0; gp < NG / 2; ++gp) {
      uint32_t x[2][4];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) ldsm4_t(x[mt], st + R::kVq + piece<D>(mt * 16 + lm_slot, gp * 2 + lm_grp));
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int gr = gp * 2 + e;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float c0[4], c1[4];
#pragma unroll
          for (int mt = 0; mt < 2; ++mt) {
            const uint32_t b0 = hmul2(pb[mt][nt][0], vsc[mt][0][gr]), b1 = hmul2(pb[mt][nt][1], vsc[mt][1][gr]);
            const uint32_t xa = x[mt][2 * e], xb = x[mt][2 * e + 1], ya = xa >> 8, yb = xb >> 8;
            if (mt == 0) {
              mma16_set(c0, xa & 0x000F000Fu, xa & 0x00F000F0u, xb & 0x000F000Fu, xb & 0x00F000F0u, b0, b1);
              mma16_set(c1, ya & 0x000F000Fu, ya & 0x00F000F0u, yb & 0x000F000Fu, yb & 0x00F000F0u, b0, b1);
            } else {
              mma16(c0, xa & 0x000F000Fu, xa & 0x00F000F0u, xb & 0x000F000Fu, xb & 0x00F000F0u, b0, b1);
              mma16(c1, ya & 0x000F000Fu, ya & 0x00F000F0u, yb & 0x000F000Fu, yb & 0x00F000F0u, b0, b1);
            }
          }
          const float k0 = corr[nt][0] * down, k1 = corr[nt][1] * down;
          float* oo = o[nt][gr];
          oo[0] = fmaf(oo[0], k0, c0[0]);
          oo[1] = fmaf(oo[1], k1, c0[1]);
          oo[2] = fmaf(oo[2], k0, c0[2]);
          oo[3] = fmaf(oo[3], k1, c0[3]);
          oo[4] = fmaf(oo[4], k0, c1[0]);
          oo[5] = fmaf(oo[5], k1, c1[1]);
          oo[6] = fmaf(oo[6], k0, c1[2]);
          oo[7] = fmaf(oo[7], k1, c1[3]);
        }
      }
    }
    __syncwarp();
  }
  cp_wait<0>();
  __syncthreads();

  // ---- the warps' rows to shared memory (over the rings): o = codes' part + zeros' part, both
  // from units of 2^14 p
  float2* sML = reinterpret_cast<float2*>(smem);
  float* sRows = reinterpret_cast<float*>(smem + W * ROWS * 8);
  const float unit = __uint_as_float((uint32_t)(127 + 10 - fe) << 23);       // 2^(24 - 14 - fe)
  constexpr float kZ = 1.f / 16384.f;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    float* row = sRows + (warp * ROWS + nt * 8 + 2 * t4) * kPad;
#pragma unroll
    for (int gr = 0; gr < NG; ++gr) {
      const float za = __shfl_sync(0xffffffffu, zl[nt][0], 4 * gr + t4) * kZ;
      const float zc = __shfl_sync(0xffffffffu, zl[nt][1], 4 * gr + t4) * kZ;
      const float* oo = o[nt][gr];
      const int d = 32 * gr + 4 * g;
      *reinterpret_cast<float4*>(row + d) =
          make_float4(fmaf(oo[0], unit, za), fmaf(oo[2], unit * 0.0625f, za), fmaf(oo[4], unit, za), fmaf(oo[6], unit * 0.0625f, za));
      *reinterpret_cast<float4*>(row + kPad + d) =
          make_float4(fmaf(oo[1], unit, zc), fmaf(oo[3], unit * 0.0625f, zc), fmaf(oo[5], unit, zc), fmaf(oo[7], unit * 0.0625f, zc));
    }
    if (g == 4) {       // the ones' row of the zero-term products: the row sums
      sML[warp * ROWS + nt * 8 + 2 * t4] = make_float2(m[nt][0] * fr[nt][0], zl[nt][0] * kZ);
      sML[warp * ROWS + nt * 8 + 2 * t4 + 1] = make_float2(m[nt][1] * fr[nt][1], zl[nt][1] * kZ);
    }
  }
  __syncthreads();
  finish<D, ROWS, W>(p, s, h, rt, blockIdx.x, W, sRows, sML, sML);
}

template <int D, int NT, int W>
constexpr size_t decode_smem() {
  const size_t ring = (size_t)W * Ring<D>::kWarpBytes;
  const size_t rows = (size_t)W * 8 * NT * ((D + 4) * 4 + 8);
  const size_t block = (size_t)W * 8 * NT * 8 + (size_t)8 * NT * (D + 4) * 4 + 2 * 32 * (D + 8) * 2;
  const size_t most = ring > rows ? ring : rows;
  return most > block ? most : block;
}

template <int D, int NT, int W, int MINB, bool FAST>
int launch(const DecodeParams& p, cudaStream_t st) {
  constexpr size_t smem = decode_smem<D, NT, W>();
  auto kernel = decode_attention_kernel<D, NT, W, MINB, FAST>;
  static bool ready[64] = {false};       // per device: the attributes are set once
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return MA_ERR_CUDA;
  if (dev < 0 || dev >= 64 || !ready[dev]) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess ||
        cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared) != cudaSuccess)
      return MA_ERR_CUDA;
    if (dev >= 0 && dev < 64) ready[dev] = true;
  }
  kernel<<<dim3(p.slots, p.H * p.row_tiles), W * 32, smem, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? MA_OK : MA_ERR_CUDA;
}

// Tiles that are contiguous in storage: positions packed back to back, K and V arrays of one
// geometry, 32-slot tiles that do not straddle pages, scale blocks on 16-byte boundaries.
bool contiguous_tiles(const ma_kv& kv, int D) {
  if (kv.mask != nullptr) return false;
  if (kv.pages != nullptr && kv.page_size % kTile != 0) return false;
  if (kv.skq[2] != D / 2 || kv.sks[2] != D / 32) return false;
  for (int i = 0; i < 3; ++i)
    if (kv.skq[i] != kv.svq[i] || kv.sks[i] != kv.svs[i] || (i < 2 && kv.sks[i] % 8 != 0)) return false;
  const uintptr_t bits = reinterpret_cast<uintptr_t>(kv.ks) | reinterpret_cast<uintptr_t>(kv.kz) |
                         reinterpret_cast<uintptr_t>(kv.vs) | reinterpret_cast<uintptr_t>(kv.vz);
  return (bits & 15) == 0;
}

int rows_per_tile(int R) { return R <= 8 ? 8 : 16; }

template <int D>
int launch_rows(const DecodeParams& p, cudaStream_t st) {
  const bool fast = contiguous_tiles(p.kv, D);
  if (rows_per_tile(p.R) == 8) return fast ? launch<D, 1, 8, 2, true>(p, st) : launch<D, 1, 8, 2, false>(p, st);
  return fast ? launch<D, 2, 8, 1, true>(p, st) : launch<D, 2, 8, 1, false>(p, st);
}

}  // namespace

// Grid: `slots` CTAs per (head, row tile) -- at most `target` equal chunks over the sequences, one
// more per sequence for its remainder, one per sequence for the block's keys.
void plan_decode(int B, int H, int R, int Tc, DecodePlan& plan) {
  plan.rows = rows_per_tile(R);
  plan.row_tiles = (R + plan.rows - 1) / plan.rows;
  const int per_head = H * plan.row_tiles;
  int target = (device_sm_count() * 6 + per_head - 1) / per_head;
  if (target < 1) target = 1;
  plan.target = target;
  plan.slots = target + B + (Tc > 0 ? B : 0);
}

int launch_decode_attention(DecodeParams& p, cudaStream_t st) {
  p.tiles_per_page = p.kv.pages != nullptr ? p.kv.page_size / kTile : 1;
  p.tile_div.set(p.tiles_per_page > 0 ? p.tiles_per_page : 1);
  return p.D == 128 ? launch_rows<128>(p, st) : launch_rows<64>(p, st);
}

}  // namespace ma
