// Page tables and slot maps of a paged cache from the requests' old and new lengths, on the
// device and in one launch.
//
// With had_b = ceil(len_b / page) and get_b = ceil(want_b / page): a shrinking request hands the
// pages get_b .. had_b - 1 back (they join the top of the free stack in (request, page) order),
// a growing one takes get_b - had_b pages from the top. Requests grow in order while the pages
// and the slot map last; from the first that does not fit on, none grows. Then every new token
// gets its slot page * page_size + offset, its request and its position.
//
// Bound: the launch at decode sizes (a few KB), HBM writes for prompts (16 B a token). Every CTA
// scans all requests itself -- 3 prefix sums of at most 8192 lengths that sit in L2 -- and
// then expands its share of the tokens and table entries, so one launch does without a wait
// between CTAs: the only thing a CTA must not do is overwrite lengths that another has yet to
// read, so the CTA that arrives last at the ticket, after its reads, writes them.
//
// Measured: 8 requests by a token each 4.8 us, 256 by 2 to 16 8.0 us (the scan's and the page look-ups'
// latency), 600 prompts of 1 to 16384 tokens 22.4 us (74 MB: 3.3 TB/s; the scan is 4 us of it).
#include "ma_kernels.cuh"

namespace ma {

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxRequests = 8192;

// a + b, or the largest value: sums only have to be right up to the limits they are held to
__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) {
  const uint32_t s = a + b;
  return s < a ? 0xffffffffu : s;
}

// Exclusive saturating scan over the CTA of three sums at once; total[] = the CTA's sums.
__device__ __forceinline__ void block_scan3(uint32_t v[3], uint32_t total[3], uint32_t (*sWarp)[kWarps]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t incl[3];
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    incl[k] = v[k];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t u = __shfl_up_sync(0xffffffffu, incl[k], o);
      if (lane >= o) incl[k] = add_sat(incl[k], u);
    }
    if (lane == 31) sWarp[k][warp] = incl[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 3; ++k) {           // every warp scans the warps' sums for itself
    uint32_t u = lane < kWarps ? sWarp[k][lane] : 0u;
#pragma unroll
    for (int o = 1; o < kWarps; o <<= 1) {
      const uint32_t x = __shfl_up_sync(0xffffffffu, u, o);
      if (lane >= o) u = add_sat(u, x);
    }
    total[k] = __shfl_sync(0xffffffffu, u, kWarps - 1);
    const uint32_t before = __shfl_sync(0xffffffffu, u, warp > 0 ? warp - 1 : 0);
    uint32_t lower = __shfl_up_sync(0xffffffffu, incl[k], 1);
    if (lane == 0) lower = 0u;
    v[k] = warp > 0 ? add_sat(lower, before) : lower;
  }
}

// The last b in [0, n) with start[b] <= x (start ascending, start[0] = 0 <= x).
__device__ __forceinline__ int owner_of(const int* start, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kThreads) page_plan_kernel(const __grid_constant__ PagePlanParams p) {
  extern __shared__ int sMem[];
  __shared__ uint32_t sWarp[3][kWarps];
  __shared__ int sLast;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, B = p.B;
  // [B + 1] first new token, first taken page, first returned page of each request; [B] old
  // length and wanted length
  int* sTok = sMem;
  int* sTake = sTok + B + 1;
  int* sGive = sTake + B + 1;
  int* sLen = sGive + B + 1;
  int* sWant = sLen + B;
  auto pages_of = [&](int len) { return len > 0 ? p.page_div.div(len - 1) + 1 : 0; };

  pdl_wait();
  pdl_launch_dependents();
  const int count = min(max(*p.free_count, 0), p.num_pages);
  const int64_t most = (int64_t)p.width * p.page_size;      // a length past its table is the table's
  const int longest = most < 0x7fffffffLL ? (int)most : 0x7fffffff;
  // ---- the sums of all requests as they ask: pages needed and tokens (saturating), pages
  // returned. A thread has `each` neighbouring requests.
  const int each = (B + kThreads - 1) / kThreads, b_lo = min(B, tid * each), b_hi = min(B, b_lo + each);
  uint32_t v[3] = {0u, 0u, 0u}, total[3];
  for (int b = b_lo; b < b_hi; ++b) {
    const int len = min(max(p.lens[b], 0), longest);
    int want = max(p.new_lens[b], 0);
    if (want > longest) want = len;        // longer than the table: stays as it is
    sLen[b] = len;
    sWant[b] = want;
    const int had = pages_of(len), get = pages_of(want);
    v[0] = add_sat(v[0], max(get - had, 0));
    v[1] = add_sat(v[1], max(want - len, 0));
    sGive[b] = (int)v[2];
    v[2] += max(had - get, 0);
    sTake[b] = (int)v[0];                  // inclusive sums of the thread's own requests, for now
    sTok[b] = (int)v[1];
  }
  block_scan3(v, total, sWarp);
  const uint32_t give0 = total[2];
  // ---- grants: the sums only grow, so the requests that fit are the first ones; behind the last of
  // them the sums stay
  const uint32_t avail = (uint32_t)count + give0;
  uint32_t taken = 0u, tokens = 0u;
  for (int b = b_lo; b < b_hi; ++b) {
    const uint32_t need = add_sat(v[0], (uint32_t)sTake[b]), tok = add_sat(v[1], (uint32_t)sTok[b]);
    sTake[b] = (int)need;
    sTok[b] = (int)tok;
    sGive[b] += (int)v[2];
    if (need <= avail && tok <= (uint32_t)p.max_tokens) {
      taken = need;
      tokens = tok;
    }
  }
  __syncthreads();                         // the scan's sums are read
  taken = __reduce_max_sync(0xffffffffu, taken);
  tokens = __reduce_max_sync(0xffffffffu, tokens);
  if (lane == 0) {
    sWarp[0][warp] = taken;
    sWarp[1][warp] = tokens;
  }
  __syncthreads();
  taken = __reduce_max_sync(0xffffffffu, lane < kWarps ? sWarp[0][lane] : 0u);
  tokens = __reduce_max_sync(0xffffffffu, lane < kWarps ? sWarp[1][lane] : 0u);
  for (int b = b_lo; b < b_hi; ++b) {             // exclusive sums of what is granted
    const int len = sLen[b], want = sWant[b];
    const bool fits = (uint32_t)sTake[b] <= avail && (uint32_t)sTok[b] <= (uint32_t)p.max_tokens;
    sTake[b] = fits ? sTake[b] - max(pages_of(want) - pages_of(len), 0) : (int)taken;
    sTok[b] = fits ? sTok[b] - max(want - len, 0) : (int)tokens;
    if (!fits && want > len) sWant[b] = len;
  }
  if (tid == 0) {
    sTake[B] = (int)taken;
    sTok[B] = (int)tokens;
    sGive[B] = (int)give0;
  }
  // (a table that gives back more pages than the pool has lost is the caller's error: the count
  // stops at the pool's size)
  const int top = count + (int)give0, left = min(top - (int)taken, p.num_pages);
  __syncthreads();                           // every length of this CTA's copy is read and granted

  if (tid == 0) {
    sLast = 1;
    if (gridDim.x > 1) {
      __threadfence();
      sLast = atomicAdd(p.ticket, 1u) == gridDim.x - 1;
      if (sLast) *p.ticket = 0u;
    }
  }
  __syncthreads();
  if (sLast) {
    for (int b = tid; b <= B; b += kThreads) {
      p.starts[b] = sTok[b];
      if (b < B) p.lens_out[b] = sWant[b];
    }
    if (tid == 0) *p.count_out = left;
  }

  // entry i of the stack after the returned pages were put on it
  auto stacked = [&](int i) -> int {
    if (i < count) return p.free_list[i];
    const int r = i - count;
    const int b = owner_of(sGive, B, r);
    return p.pages[(int64_t)b * p.spg + pages_of(sWant[b]) + (r - sGive[b])];
  };
  auto taken_page = [&](int b, int k) -> int { return stacked(top - 1 - (sTake[b] + k)); };

  const int64_t step = (int64_t)gridDim.x * kThreads, first = (int64_t)blockIdx.x * kThreads + tid;

  // ---- the tokens, four to a thread and a run of them to a warp, so that a lane's next four are
  // mostly of the same request
  const int64_t quads = ((int64_t)p.max_tokens + 3) / 4, all_warps = (int64_t)gridDim.x * kWarps;
  const int64_t run = ((quads + all_warps - 1) / all_warps + 31) / 32 * 32, at_warp = (int64_t)blockIdx.x * kWarps + warp;
  const int64_t run_end = min(quads, (at_warp + 1) * run);
  int b = -1;
  for (int64_t qd = at_warp * run + lane; qd < run_end; qd += 32) {
    const int i0 = (int)(qd * 4);
    long long slot[4];
    int own[4], pos[4];
    // requests without tokens share their start with the next: the owner is the last one at or below
    if (i0 < (int)tokens && (b < 0 || i0 >= sTok[b + 1])) b = owner_of(sTok, B, i0);
    auto page_at = [&](int at) {
      const int had = pages_of(sLen[b]);
      const int page = at < had ? p.pages[(int64_t)b * p.spg + at] : taken_page(b, at - had);
      return page >= 0 && page < p.num_pages ? page : -1;
    };
    const int x0 = i0 < (int)tokens ? sLen[b] + (i0 - sTok[b]) : 0;
    int at = p.page_div.div(x0), off = x0 - at * p.page_size;
    if (i0 < (int)tokens && i0 + 3 < sTok[b + 1] && p.page_size >= 4) {
      // one request, at most two pages (some lane of a warp crosses one in most rounds)
      const int page = page_at(at), left_here = p.page_size - off;
      const int after = left_here < 4 ? page_at(at + 1) : -1;
      const long long here = page >= 0 ? (long long)page * p.page_size + off : -1ll;
      const long long there = after >= 0 ? (long long)after * p.page_size - left_here : -1ll;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        slot[e] = e < left_here ? (page >= 0 ? here + e : -1ll) : (after >= 0 ? there + e : -1ll);
        own[e] = b;
        pos[e] = x0 + e;
      }
    } else {
      int page = -2;
#pragma unroll 1
      for (int e = 0; e < 4; ++e) {
        const int i = i0 + e;
        long long s = -1;
        int o = -1, x = -1;
        if (i < (int)tokens) {
          if (i >= sTok[b + 1]) {
            do ++b; while (i >= sTok[b + 1]);
            page = -2;
          }
          x = sLen[b] + (i - sTok[b]);
          at = p.page_div.div(x);
          off = x - at * p.page_size;
          if (page == -2 || off == 0) page = page_at(at);
          o = b;
          if (page >= 0) s = (long long)page * p.page_size + off;
        }
        // (registers, not local memory: no dynamic index)
        if (e == 0) { slot[0] = s; own[0] = o; pos[0] = x; }
        else if (e == 1) { slot[1] = s; own[1] = o; pos[1] = x; }
        else if (e == 2) { slot[2] = s; own[2] = o; pos[2] = x; }
        else { slot[3] = s; own[3] = o; pos[3] = x; }
      }
    }
    if (i0 + 4 <= p.max_tokens) {
      reinterpret_cast<longlong2*>(p.slots + i0)[0] = make_longlong2(slot[0], slot[1]);
      reinterpret_cast<longlong2*>(p.slots + i0)[1] = make_longlong2(slot[2], slot[3]);
      *reinterpret_cast<int4*>(p.seqs + i0) = make_int4(own[0], own[1], own[2], own[3]);
      *reinterpret_cast<int4*>(p.positions + i0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i0 + e < p.max_tokens) {
          p.slots[i0 + e] = slot[e];
          p.seqs[i0 + e] = own[e];
          p.positions[i0 + e] = pos[e];
        }
    }
  }

  // ---- the page table, 32 entries of a request per warp and round. In place only the taken pages
  // are written; returned entries keep their stale number behind the length, so nothing that is
  // read here is written here.
  const int warps = gridDim.x * kWarps, pieces = (p.width + 31) / 32;
  for (int64_t u = blockIdx.x * kWarps + warp; u < (int64_t)B * pieces; u += warps) {
    const int r = (int)(u / pieces), j0 = (int)(u - (int64_t)r * pieces) * 32;
    const int had = pages_of(sLen[r]), taken_r = sTake[r + 1] - sTake[r];
    if (p.pages_in_place && (j0 + 32 <= had || j0 >= had + taken_r)) continue;
    const int j = j0 + lane, k = j - had;
    if (j >= p.width) continue;
    if (k >= 0 && k < taken_r) p.pages_out[(int64_t)r * p.spg_out + j] = taken_page(r, k);
    else if (!p.pages_in_place) p.pages_out[(int64_t)r * p.spg_out + j] = p.pages[(int64_t)r * p.spg + j];
  }

  // ---- the free stack: the returned pages that were not taken again
  if (p.free_in_place) {
    for (int64_t i = count + first; i < left; i += step) p.free_out[i] = stacked((int)i);
  } else {
    for (int64_t i = first; i < p.num_pages; i += step)
      p.free_out[i] = i >= count && i < left ? stacked((int)i) : p.free_list[i];
  }
}

// The pages that are in the pool, moved to the front of each request's table in their order, a warp
// per request; lens_out counts their slots. A copy of the cache by this table has no dead slot below
// its lengths, which a copy in place of the slots would have to mask.
constexpr int kLiveWarps = 4;

__global__ void __launch_bounds__(kLiveWarps * 32) live_pages_kernel(const ma_kv kv, int B, int width, int32_t* pages_out,
                                                                      int32_t* lens_out) {
  const int lane = threadIdx.x & 31, b = blockIdx.x * kLiveWarps + (threadIdx.x >> 5);
  pdl_wait();
  pdl_launch_dependents();
  if (b >= B) return;
  int n = kv.nq;
  if (kv.lens != nullptr) n = min(n, max(kv.lens[b], 0));
  const int had = (int)(((int64_t)n + kv.page_size - 1) / kv.page_size);
  int32_t* out = pages_out + (int64_t)b * width;
  int count = 0;
  bool last = false;
  for (int j0 = 0; j0 < had; j0 += 32) {
    const int j = j0 + lane, page = j < had ? kv.pages[(int64_t)b * kv.spg + j] : -1;
    const unsigned live = __ballot_sync(0xffffffffu, page >= 0 && page < kv.num_pages);
    if (live >> lane & 1u) out[count + __popc(live & ((1u << lane) - 1u))] = page;
    count += __popc(live);
    if (had - j0 <= 32) last = live >> (had - 1 - j0) & 1u;
  }
  for (int j = count + lane; j < width; j += 32) out[j] = -1;
  if (lane == 0) lens_out[b] = (int)((int64_t)count * kv.page_size - (last ? (int64_t)had * kv.page_size - n : 0));
}

}  // namespace

int launch_live_pages(const ma_kv& kv, int B, int32_t* pages_out, int32_t* lens_out, cudaStream_t st) {
  const int width = (int)(((int64_t)kv.nq + kv.page_size - 1) / kv.page_size);
  return launch_pdl(live_pages_kernel, dim3((unsigned)((B + kLiveWarps - 1) / kLiveWarps)), dim3(kLiveWarps * 32), 0, st, kv, B,
                    width, pages_out, lens_out) == cudaSuccess ? MA_OK : MA_ERR_CUDA;
}

int page_plan_max_requests() { return kMaxRequests; }

int launch_page_plan(PagePlanParams& p, cudaStream_t st) {
  // what the largest call takes is opted in to once per device: the default limit of 48 KB holds for
  // the dynamic bytes and the kernel's static ones together
  constexpr size_t kMost = (5 * (size_t)kMaxRequests + 3) * sizeof(int);
  static bool ready[64] = {false};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return MA_ERR_CUDA;
  if (dev < 0 || dev >= 64 || !ready[dev]) {
    if (cudaFuncSetAttribute(page_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMost) != cudaSuccess)
      return MA_ERR_CUDA;
    if (dev >= 0 && dev < 64) ready[dev] = true;
  }
  const size_t smem = (5 * (size_t)p.B + 3) * sizeof(int);
  int64_t items = ((int64_t)p.max_tokens + 3) / 4;
  if (!p.pages_in_place) items = items > (int64_t)p.B * p.width ? items : (int64_t)p.B * p.width;
  if (!p.free_in_place) items = items > p.num_pages ? items : p.num_pages;
  int64_t grid = (items + kThreads - 1) / kThreads;
  const int64_t cap = (int64_t)device_sm_count() * (p.B <= 1024 ? 2 : 1);
  p.page_div.set((uint32_t)p.page_size);
  grid = grid < 1 ? 1 : grid > cap ? cap : grid;
  return launch_pdl(page_plan_kernel, dim3((unsigned)grid), dim3(kThreads), smem, st, p) == cudaSuccess ? MA_OK : MA_ERR_CUDA;
}

}  // namespace ma
