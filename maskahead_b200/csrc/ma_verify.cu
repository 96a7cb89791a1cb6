// Drafted tokens against the target's probabilities: the accepted run of each request and the
// token drawn after it, from given uniforms.
//
// Draft i of a request is accepted while u_i q_i(x_i) < p_i(x_i); with a drafts accepted the next
// token is drawn from max(p_a - q_a, 0), or from p_a itself when every draft was accepted. The
// drawing inverts the cumulative sum in whole numbers: w_v = floor(min(r_v, 1) 2^40), threshold
// floor(total floor(u 2^24) / 2^24), first v whose inclusive sum is above it. Sums of whole
// numbers do not depend on their order, so the token does not depend on the split.
//
// Bound: HBM, one row of p and one of q per request (the other rows are read at one element
// each). A warp sums one span of one request's row; the last CTA of the request to arrive
// finds the span that holds the threshold and rescans that span alone, from L2. The spans make
// about one wave of CTAs, because every CTA first finds the accepted run for itself (two
// dependent loads, 1.5 us).
//
// floor(r 2^40) takes no conversion (those run at an eighth of the FMA rate): with t = r 2^20 +
// 2^23 truncated, t's low bits are the upper 20 bits of the weight, and the remainder gives the
// lower 20 in the same way; the two halves are summed as 32-bit whole numbers.
#include "ma_kernels.cuh"

namespace ma {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxSpans = 1024;
constexpr int kMaxSpan = 4096;          // elements: what the last CTA rescans
constexpr int kMaxRequests = 65535;
constexpr uint32_t kMagicBits = 0x4B000000u;       // 2^23

__device__ __forceinline__ float value(const float* p, int64_t i) { return __ldg(p + i); }
__device__ __forceinline__ float value(const __nv_bfloat16* p, int64_t i) { return __bfloat162float(p[i]); }
__device__ __forceinline__ float value(const __half* p, int64_t i) { return __half2float(p[i]); }

// The halves of floor(r 2^40), r in [0, 1], each plus the bits of 2^23.
__device__ __forceinline__ void weight_halves(float r, uint32_t& hi, uint32_t& lo) {
  const float t = __fmaf_rz(r, 1048576.f, 8388608.f);
  const float rest = __fmaf_rn(r, 1048576.f, -(t - 8388608.f));      // exact
  hi = __float_as_uint(t);
  lo = __float_as_uint(__fmaf_rz(rest, 1048576.f, 8388608.f));
}
__device__ __forceinline__ unsigned long long join(uint32_t hi, uint32_t lo, uint32_t n) {
  return ((unsigned long long)(hi - n * kMagicBits) << 20) + (lo - n * kMagicBits);
}

__device__ __forceinline__ unsigned long long warp_sum64(unsigned long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Inclusive scan over the CTA; returns the CTA's sum in `total`.
__device__ __forceinline__ unsigned long long block_scan(unsigned long long v, unsigned long long& total,
                                                         unsigned long long* sWarp) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  __syncthreads();
  if (lane == 31) sWarp[warp] = v;
  __syncthreads();
  unsigned long long before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    const unsigned long long u = sWarp[w];
    if (w < warp) before += u;
    total += u;
  }
  return v + before;
}

// The row the next token is drawn from: p, and q to subtract (null: nothing; dropped >= 0:
// a one-hot draft, that token's weight is 0). Saturation clamps to [0, 1] and takes NaN to 0.
template <typename T>
struct Row {
  const T *p, *q;
  int dropped;
  __device__ __forceinline__ float rest(int v) const {
    const float a = value(p, v);
    return __saturatef(q != nullptr ? a - value(q, v) : a);
  }
  __device__ __forceinline__ unsigned long long operator()(int v) const {
    uint32_t hi, lo;
    weight_halves(rest(v), hi, lo);
    return v == dropped ? 0ull : join(hi, lo, 1);
  }
  // the sum over [begin, end) by one warp: at most kMaxSpan elements, 128 a lane
  template <bool Q>
  __device__ __forceinline__ unsigned long long span(int begin, int end) const {
    const int lane = threadIdx.x & 31;
    uint32_t hi = 0u, lo = 0u, n = 0u;
    int v = begin + lane;
    for (; v + 7 * 32 < end; v += 8 * 32, n += 8) {
      float a[8], b[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        a[e] = value(p, v + e * 32);
        b[e] = Q ? value(q, v + e * 32) : 0.f;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        uint32_t x, y;
        weight_halves(__saturatef(a[e] - b[e]), x, y);
        hi += x;
        lo += y;
      }
    }
    for (; v < end; v += 32, ++n) {
      uint32_t x, y;
      weight_halves(rest(v), x, y);
      hi += x;
      lo += y;
    }
    unsigned long long s = join(hi, lo, n);
    if (dropped >= begin && dropped < end && ((dropped - begin) & 31) == lane) {      // the lane that counted it
      uint32_t x, y;
      weight_halves(rest(dropped), x, y);
      s -= join(x, y, 1);
    }
    return warp_sum64(s);
  }
  __device__ __forceinline__ unsigned long long span(int begin, int end) const {
    return q != nullptr ? span<true>(begin, end) : span<false>(begin, end);
  }
};

// The first element of [begin, end) whose inclusive sum (from `before`) is above the mark, by the
// whole CTA, kMaxSpan elements at a time; -1 when there is none.
template <typename T>
__device__ int find_crossing(const Row<T>& row, int begin, int end, unsigned long long before, unsigned long long mark,
                             unsigned long long* sWarp, int* sFound) {
  constexpr int kEach = kMaxSpan / kThreads;
  for (int v0 = begin; v0 < end; v0 += kMaxSpan) {
    const int per = min(kEach, (end - v0 + kThreads - 1) / kThreads);       // consecutive elements of a thread
    unsigned long long w[kEach], mine = 0, total;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const int v = v0 + threadIdx.x * per + e;
      w[e] = e < per && v < end ? row(v) : 0ull;
      mine += w[e];
    }
    const unsigned long long incl = before + block_scan(mine, total, sWarp);
    if (threadIdx.x == 0) *sFound = -1;
    __syncthreads();
    if (incl > mark && incl - mine <= mark) {                // exactly one thread
      unsigned long long at = incl - mine;
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        if (at <= mark && at + w[e] > mark) *sFound = v0 + threadIdx.x * per + e;
        at += w[e];
      }
    }
    __syncthreads();
    const int found = *sFound;
    if (found >= 0) return found;
    before += total;
  }
  return -1;
}

__device__ __forceinline__ unsigned long long mark_of(unsigned long long total, float u) {
  const unsigned long long k = (unsigned long long)fminf(fmaxf(u * 16777216.f, 0.f), 16777215.f);
  return (total >> 24) * k + (((total & 0xffffffull) * k) >> 24);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) verify_kernel(const __grid_constant__ VerifyParams p) {
  __shared__ unsigned long long sWarp[kWarps];
  __shared__ int sRun, sLast, sFound, sSpan;
  __shared__ unsigned long long sBefore;
  const int b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T* target = reinterpret_cast<const T*>(p.target) + (int64_t)b * p.st[0];
  const T* draft = p.draft == nullptr ? nullptr : reinterpret_cast<const T*>(p.draft) + (int64_t)b * p.sd[0];
  const int n = min(max(p.counts == nullptr ? p.K : p.counts[b], 0), p.K);
  if (warp == 0) {       // the accepted run: the first refused draft, 32 at a time
    int run = n;
    for (int i0 = 0; i0 < n; i0 += 32) {
      const int i = i0 + lane;
      bool good = true;
      if (i < n) {
        const int x = p.tokens[(int64_t)b * p.K + i];
        good = false;
        if (x >= 0 && x < p.V) {
          const float q = draft == nullptr ? 1.f : value(draft, (int64_t)i * p.sd[1] + x);
          good = p.uniforms[(int64_t)b * (p.K + 1) + i] * q < value(target, (int64_t)i * p.st[1] + x);
        }
      }
      const unsigned bad = ~__ballot_sync(0xffffffffu, good);
      if (bad) {
        run = i0 + __ffs(bad) - 1;
        break;
      }
    }
    if (lane == 0) sRun = run;
  }
  __syncthreads();
  const int run = sRun;
  Row<T> row;
  row.p = target + (int64_t)run * p.st[1];
  row.q = run < n && draft != nullptr ? draft + (int64_t)run * p.sd[1] : nullptr;
  row.dropped = run < n && draft == nullptr ? p.tokens[(int64_t)b * p.K + run] : -1;

  // ---- a span per warp
  unsigned long long* sums = p.sums + (int64_t)b * p.spans;
  const int own = blockIdx.x * kWarps + warp;
  if (own < p.spans) {
    const unsigned long long sum = row.span(own * p.span, min(p.V, (own + 1) * p.span));
    if (lane == 0) __stcg(&sums[own], sum);
  }
  __threadfence();
  __syncthreads();
  if (tid == 0) {
    sLast = atomicAdd(&p.tickets[b], 1u) == gridDim.x - 1;
    if (sLast) p.tickets[b] = 0u;
  }
  __syncthreads();
  if (!sLast) return;
  __threadfence();

  // ---- the request's last CTA: the span that holds the threshold, then the token
  constexpr int kEach = kMaxSpans / kThreads;
  unsigned long long v[kEach], mine = 0, total;
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int c = tid * kEach + e;
    v[e] = c < p.spans ? __ldcg(&sums[c]) : 0ull;
    mine += v[e];
  }
  const unsigned long long incl = block_scan(mine, total, sWarp);
  const float u = p.uniforms[(int64_t)b * (p.K + 1) + p.K];
  int token = -1;
  if (total > 0) {
    const unsigned long long mark = mark_of(total, u);
    unsigned long long at = incl - mine;
    if (incl > mark && at <= mark) {        // exactly one thread
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        if (at <= mark && at + v[e] > mark) {
          sSpan = tid * kEach + e;
          sBefore = at;
        }
        at += v[e];
      }
    }
    __syncthreads();
    token = find_crossing(row, sSpan * p.span, min(p.V, (sSpan + 1) * p.span), sBefore, mark, sWarp, &sFound);
  } else {
    // no residual mass (p <= q everywhere): the row of p itself, read again whole
    row.q = nullptr;
    row.dropped = -1;
    unsigned long long s = 0;
    for (int x = tid; x < p.V; x += kThreads) s += row(x);
    block_scan(s, total, sWarp);
    if (total > 0) token = find_crossing(row, 0, p.V, 0ull, mark_of(total, u), sWarp, &sFound);
  }
  if (tid == 0) p.accepted[b] = run;
  for (int i = tid; i <= p.K; i += kThreads)
    p.out[(int64_t)b * (p.K + 1) + i] = i < run ? p.tokens[(int64_t)b * p.K + i] : i == run ? token : -1;
}

}  // namespace

int verify_max_requests() { return kMaxRequests; }

// Elements per span: about one wave of CTAs (5 an SM) over all requests, in steps of the 256
// elements that a warp loads at once; at most kMaxSpans spans a row.
void plan_verify(int B, int V, int& span, int& spans) {
  const int64_t warps = (int64_t)device_sm_count() * 5 * kWarps;
  int64_t n = ((int64_t)B * V + warps - 1) / warps;
  n = (n + 255) / 256 * 256;
  if (n > kMaxSpan) n = kMaxSpan;
  while ((V + n - 1) / n > kMaxSpans) n += 256;
  span = (int)n;
  spans = (int)((V + n - 1) / n);
}

int launch_verify_drafts(const VerifyParams& p, int dtype, cudaStream_t st) {
  const dim3 grid((p.spans + kWarps - 1) / kWarps, p.B);
  if (dtype == MA_F32) verify_kernel<float><<<grid, kThreads, 0, st>>>(p);
  else if (dtype == MA_BF16) verify_kernel<__nv_bfloat16><<<grid, kThreads, 0, st>>>(p);
  else verify_kernel<__half><<<grid, kThreads, 0, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? MA_OK : MA_ERR_CUDA;
}

}  // namespace ma
