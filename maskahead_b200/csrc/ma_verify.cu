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
// each). A CTA sums one chunk of one request's row; the last CTA of the request to arrive
// finds the chunk that holds the threshold and rescans that chunk alone, from L2.
#include "ma_kernels.cuh"

namespace ma {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxChunks = 1024;
constexpr int kMaxRequests = 65535;

__device__ __forceinline__ float value(const float* p, int64_t i) { return __ldg(p + i); }
__device__ __forceinline__ float value(const __nv_bfloat16* p, int64_t i) { return __bfloat162float(p[i]); }
__device__ __forceinline__ float value(const __half* p, int64_t i) { return __half2float(p[i]); }

// floor(min(r, 1) 2^40) of a positive r, 0 otherwise (and for NaN)
__device__ __forceinline__ unsigned long long weight(float r) {
  return r > 0.f ? __float2ull_rz(fminf(r, 1.f) * 1099511627776.f) : 0ull;
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
// a one-hot draft, that token's weight is 0).
template <typename T>
struct Row {
  const T *p, *q;
  int dropped;
  __device__ __forceinline__ unsigned long long operator()(int v) const {
    const float a = value(p, v);
    const unsigned long long w = weight(q != nullptr ? a - value(q, v) : a);
    return v == dropped ? 0ull : w;
  }
};

// The first element of [begin, end) whose inclusive sum (from `before`) is above the mark, by the
// whole CTA; -1 when there is none. sums: this CTA's shared scratch.
template <typename T>
__device__ int find_crossing(const Row<T>& row, int begin, int end, unsigned long long before, unsigned long long mark,
                             unsigned long long* sWarp, int* sFound) {
  for (int v0 = begin; v0 < end; v0 += kThreads) {
    const int v = v0 + threadIdx.x;
    const unsigned long long w = v < end ? row(v) : 0ull;
    unsigned long long total;
    const unsigned long long incl = before + block_scan(w, total, sWarp);
    if (threadIdx.x == 0) *sFound = -1;
    __syncthreads();
    if (incl > mark && incl - w <= mark) *sFound = v;     // exactly one thread
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
  __shared__ int sRun, sLast, sFound, sChunk;
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

  const int begin = blockIdx.x * p.chunk, end = min(p.V, begin + p.chunk);
  unsigned long long sum = 0;
#pragma unroll 8
  for (int v = begin + tid; v < end; v += kThreads) sum += row(v);
  sum = warp_sum64(sum);
  if (lane == 0) sWarp[warp] = sum;
  __syncthreads();
  unsigned long long* sums = p.sums + (int64_t)b * p.chunks;
  if (tid == 0) {
    sum = 0;
    for (int w = 0; w < kWarps; ++w) sum += sWarp[w];
    __stcg(&sums[blockIdx.x], sum);
    __threadfence();
    sLast = atomicAdd(&p.tickets[b], 1u) == gridDim.x - 1;
    if (sLast) p.tickets[b] = 0u;
  }
  __syncthreads();
  if (!sLast) return;
  __threadfence();

  // ---- the request's last CTA: the chunk that holds the threshold, then the token
  unsigned long long v[kMaxChunks / kThreads], mine = 0, total;
#pragma unroll
  for (int e = 0; e < kMaxChunks / kThreads; ++e) {
    const int c = tid * (kMaxChunks / kThreads) + e;
    v[e] = c < p.chunks ? __ldcg(&sums[c]) : 0ull;
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
      for (int e = 0; e < kMaxChunks / kThreads; ++e) {
        if (at <= mark && at + v[e] > mark) {
          sChunk = tid * (kMaxChunks / kThreads) + e;
          sBefore = at;
        }
        at += v[e];
      }
    }
    __syncthreads();
    const int c0 = sChunk * p.chunk;
    token = find_crossing(row, c0, min(p.V, c0 + p.chunk), sBefore, mark, sWarp, &sFound);
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

// Chunks of a row: enough CTAs for the GPU when there are few requests, long enough that their
// sums stay few.
void plan_verify(int B, int V, int& chunk, int& chunks) {
  chunk = 1024;
  while (chunk < 8192 && (int64_t)B * ((V + chunk - 1) / chunk) > (int64_t)device_sm_count() * 16) chunk *= 2;
  while ((V + chunk - 1) / chunk > kMaxChunks) chunk *= 2;
  chunks = (V + chunk - 1) / chunk;
}

int launch_verify_drafts(const VerifyParams& p, int dtype, cudaStream_t st) {
  const dim3 grid(p.chunks, p.B);
  if (dtype == MA_F32) verify_kernel<float><<<grid, kThreads, 0, st>>>(p);
  else if (dtype == MA_BF16) verify_kernel<__nv_bfloat16><<<grid, kThreads, 0, st>>>(p);
  else verify_kernel<__half><<<grid, kThreads, 0, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? MA_OK : MA_ERR_CUDA;
}

}  // namespace ma
