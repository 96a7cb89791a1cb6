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
#include "ma_kernels.cuh"

namespace ma {

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxRequests = 8192;

__device__ __forceinline__ int pages_of(int len, int page) { return len / page + (len % page != 0); }

// Inclusive scan over the CTA of three sums at once; total[] = the CTA's sums.
__device__ __forceinline__ void block_scan3(long long v[3], long long total[3], long long (*sWarp)[kWarps]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int k = 0; k < 3; ++k) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long u = __shfl_up_sync(0xffffffffu, v[k], o);
      if (lane >= o) v[k] += u;
    }
    if (lane == 31) sWarp[k][warp] = v[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    long long before = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const long long u = sWarp[k][w];
      if (w < warp) before += u;
      sum += u;
    }
    v[k] += before;
    total[k] = sum;
  }
  __syncthreads();
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
  __shared__ long long sWarp[3][kWarps];
  __shared__ int sLast;
  const int tid = threadIdx.x, B = p.B;
  // [B + 1] first new token, first taken page, first returned page of each request; [B] old
  // length and wanted length
  int* sTok = sMem;
  int* sTake = sTok + B + 1;
  int* sGive = sTake + B + 1;
  int* sLen = sGive + B + 1;
  int* sWant = sLen + B;

  const int count = min(max(*p.free_count, 0), p.num_pages);
  const int64_t most = (int64_t)p.width * p.page_size;      // a length past its table is the table's
  const int longest = most < 0x7fffffffLL ? (int)most : 0x7fffffff;
  long long given = 0;                      // pages handed back by all requests
  for (int b = tid; b < B; b += kThreads) {
    const int len = min(max(p.lens[b], 0), longest);
    int want = max(p.new_lens[b], 0);
    if (pages_of(want, p.page_size) > p.width) want = len;      // longer than the table: stays as it is
    sLen[b] = len;
    sWant[b] = want;
    given += max(pages_of(len, p.page_size) - pages_of(want, p.page_size), 0);
  }
  {
    long long v[3] = {given, 0, 0}, total[3];
    block_scan3(v, total, sWarp);
    given = total[0];
  }
  const long long avail = count + given;
  long long need0 = 0, tok0 = 0, give0 = 0, need_ok = 0, tok_ok = 0;
  for (int b0 = 0; b0 < B; b0 += kThreads) {
    const int b = b0 + tid;
    const int len = b < B ? sLen[b] : 0, want = b < B ? sWant[b] : 0;
    const int had = pages_of(len, p.page_size), get = pages_of(want, p.page_size);
    long long v[3] = {max(get - had, 0), max(want - len, 0), max(had - get, 0)}, total[3];
    const long long need = v[0], tok = v[1], give = v[2];
    block_scan3(v, total, sWarp);
    // the sums only grow: once one is too large no later request fits
    const bool fits = need0 + v[0] <= avail && tok0 + v[1] <= p.max_tokens;
    // exclusive sums over the granted requests: the raw ones while they fit, the last fitting
    // ones from then on
    long long ok[3] = {fits ? need : 0, fits ? tok : 0, 0}, okt[3];
    block_scan3(ok, okt, sWarp);
    if (b < B) {
      sTake[b] = (int)(need_ok + ok[0] - (fits ? need : 0));
      sTok[b] = (int)(tok_ok + ok[1] - (fits ? tok : 0));
      sGive[b] = (int)(give0 + v[2] - give);
      if (!fits && want > len) sWant[b] = len;
    }
    need0 += total[0];
    tok0 += total[1];
    give0 += total[2];
    need_ok += okt[0];
    tok_ok += okt[1];
  }
  const int taken = (int)need_ok, tokens = (int)tok_ok, back = (int)give0;
  if (tid == 0) {
    sTake[B] = taken;
    sTok[B] = tokens;
    sGive[B] = back;
  }
  // (a table that gives back more pages than the pool has lost is the caller's error: the count
  // stops at the pool's size)
  const int top = count + back, left = min(top - taken, p.num_pages);
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
    return p.pages[(int64_t)b * p.spg + pages_of(sWant[b], p.page_size) + (r - sGive[b])];
  };
  auto taken_page = [&](int b, int k) -> int { return stacked(top - 1 - (sTake[b] + k)); };

  const int64_t step = (int64_t)gridDim.x * kThreads, first = (int64_t)blockIdx.x * kThreads + tid;

  // ---- the tokens, four to a thread
  const int64_t quads = ((int64_t)p.max_tokens + 3) / 4;
  for (int64_t qd = first; qd < quads; qd += step) {
    const int i0 = (int)(qd * 4);
    long long slot[4];
    int own[4], pos[4];
    int b = -1, page = -1, at = -1, off = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = i0 + e;
      slot[e] = -1;
      own[e] = pos[e] = -1;
      if (i >= tokens) continue;
      if (b < 0 || i >= sTok[b + 1]) {
        // requests without tokens share their start with the next: the last one at or below i
        b = b < 0 ? owner_of(sTok, B, i) : b + 1;
        while (i >= sTok[b + 1]) ++b;
        at = -1;
      }
      const int x = sLen[b] + (i - sTok[b]);
      if (at < 0 || ++off == p.page_size) {
        at = x / p.page_size;
        off = x - at * p.page_size;
        const int had = pages_of(sLen[b], p.page_size);
        page = at < had ? p.pages[(int64_t)b * p.spg + at] : taken_page(b, at - had);
      }
      own[e] = b;
      pos[e] = x;
      if (page >= 0 && page < p.num_pages) slot[e] = (long long)page * p.page_size + off;
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

  // ---- the page table. In place only the taken pages are written; returned entries keep their
  // stale number behind the length, so nothing that is read here is written here.
  if (p.pages_in_place) {
    for (int64_t i = first; i < taken; i += step) {
      const int b = owner_of(sTake, B, (int)i);
      const int k = (int)i - sTake[b];
      p.pages_out[(int64_t)b * p.spg_out + pages_of(sLen[b], p.page_size) + k] = taken_page(b, k);
    }
  } else {
    const int64_t entries = (int64_t)B * p.width;
    for (int64_t i = first; i < entries; i += step) {
      const int b = (int)(i / p.width), j = (int)(i - (int64_t)b * p.width);
      const int k = j - pages_of(sLen[b], p.page_size);
      p.pages_out[(int64_t)b * p.spg_out + j] =
          k >= 0 && k < sTake[b + 1] - sTake[b] ? taken_page(b, k) : p.pages[(int64_t)b * p.spg + j];
    }
  }

  // ---- the free stack: the returned pages that were not taken again
  if (p.free_in_place) {
    for (int64_t i = count + first; i < left; i += step) p.free_out[i] = stacked((int)i);
  } else {
    for (int64_t i = first; i < p.num_pages; i += step)
      p.free_out[i] = i >= count && i < left ? stacked((int)i) : p.free_list[i];
  }
}

}  // namespace

int page_plan_max_requests() { return kMaxRequests; }

int launch_page_plan(const PagePlanParams& p, cudaStream_t st) {
  const size_t smem = (5 * (size_t)p.B + 3) * sizeof(int);
  if (cudaFuncSetAttribute(page_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 5 * (kMaxRequests + 1) * (int)sizeof(int)) !=
      cudaSuccess)
    return MA_ERR_CUDA;
  int64_t items = ((int64_t)p.max_tokens + 3) / 4;
  if (!p.pages_in_place) items = items > (int64_t)p.B * p.width ? items : (int64_t)p.B * p.width;
  if (!p.free_in_place) items = items > p.num_pages ? items : p.num_pages;
  int64_t grid = (items + kThreads - 1) / kThreads;
  const int64_t cap = (int64_t)device_sm_count() * (p.B <= 1024 ? 2 : 1);
  grid = grid < 1 ? 1 : grid > cap ? cap : grid;
  page_plan_kernel<<<(int)grid, kThreads, smem, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? MA_OK : MA_ERR_CUDA;
}

}  // namespace ma
