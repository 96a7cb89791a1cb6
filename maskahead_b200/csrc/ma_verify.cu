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
// each). A warp sums its share of a request's row in spans of 2 KB, which cp.async brings into its
// own ring of shared memory by 16-byte pieces -- rows of an odd vocabulary in 16 bits lie on any
// even address, and element loads kept too few bytes in flight (800 rows of 100003: 116 us against
// 58). The last CTA of the request to arrive finds the span that holds the threshold and rescans that
// span alone, from L2. Each CTA first finds the accepted run for itself (two dependent loads, 1.5 us).
//
// Measured: 200 requests x 5 drafts, 100003 entries in bf16, 21 us (62 MB: 2.9 TB/s; 5 us are the chain of
// dependent steps, and a request that refuses a draft reads twice the bytes of one that does not, in as many
// CTAs); 1 request x 4 drafts, 32000 in 32 bits, 5.6 us, the chain.
//
// floor(r 2^40) takes no conversion (those run at an eighth of the FMA rate): with t = r 2^20 +
// 2^23 truncated, t's low bits are the upper 20 bits of the weight, and the remainder gives the
// lower 20 in the same way; the two halves are summed as 32-bit whole numbers.
#include <type_traits>

#include "ma_kernels.cuh"

namespace ma {

namespace {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxSpans = 2048;
constexpr int kSpanBytes = 2048;        // of a span of p or q: what a warp copies at once, and the last CTA rescans
constexpr int kStages = 2;
constexpr int kBuffer = kSpanBytes + 16;                        // a span from the 16-byte boundary at or before it
constexpr int kRingBytes = kWarps * kStages * 2 * kBuffer;
constexpr int kMaxRequests = 65535;
constexpr uint32_t kMagicBits = 0x4B000000u;       // 2^23

__device__ __forceinline__ float value_of(float x) { return x; }
__device__ __forceinline__ float value_of(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float value_of(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ float value(const T* p, int64_t i) { return value_of(p[i]); }

// The halves of floor(r 2^40), r in [0, 1], each plus the bits of 2^23.
__device__ __forceinline__ void weight_halves(float r, uint32_t& hi, uint32_t& lo) {
  const float t = __fmaf_rz(r, 1048576.f, 8388608.f);
  const float rest = __fmaf_rn(r, 1048576.f, -(t - 8388608.f));      // exact
  hi = __float_as_uint(t);
  lo = __float_as_uint(__fmaf_rz(rest, 1048576.f, 8388608.f));
}
// The same for two elements in packed operations, added to the sums.
__device__ __forceinline__ void add_weights(float r0, float r1, uint32_t& hi, uint32_t& lo) {
  uint32_t t0, t1, u0, u1;
  asm("{\n.reg .b64 r, t, n, s, m;\n"
      "mov.b64 r, {%4, %5};\nmov.b64 s, {%6, %6};\nmov.b64 m, {%7, %7};\nmov.b64 n, {%8, %8};\n"
      "fma.rz.f32x2 t, r, s, m;\n"
      "fma.rn.f32x2 n, t, n, m;\n"            // 2^23 - t
      "fma.rn.f32x2 n, r, s, n;\n"            // what t leaves of r 2^20, exact
      "fma.rz.f32x2 n, n, s, m;\n"
      "mov.b64 {%0, %1}, t;\nmov.b64 {%2, %3}, n;\n}\n"
      : "=r"(t0), "=r"(t1), "=r"(u0), "=r"(u1)
      : "f"(r0), "f"(r1), "f"(1048576.f), "f"(8388608.f), "f"(-1.f));
  hi += t0 + t1;
  lo += u0 + u1;
}
__device__ __forceinline__ float2 pair_of(uint32_t w, __nv_bfloat16) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ float2 pair_of(uint32_t w, __half) { return __half22float2(*reinterpret_cast<__half2*>(&w)); }
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
};

// Elements [begin, end) of a row to shared memory, by one warp, from the 16-byte boundary at or
// before the first; returns how many bytes that is before it. (The bytes before a row are of its
// tensor's storage; nothing past `end` is read.)
template <typename T>
__device__ __forceinline__ void copy_span(uint32_t dst, const T* row, int begin, int end) {
  const uintptr_t first = reinterpret_cast<uintptr_t>(row + begin), last = reinterpret_cast<uintptr_t>(row + end);
  uintptr_t at = (first & ~uintptr_t(15)) + (threadIdx.x & 31) * 16;
#pragma unroll
  for (int e = 0; e < (kBuffer + 511) / 512; ++e, at += 512) {
    if (at < last) {
      const uint32_t bytes = (uint32_t)(last - at < 16 ? last - at : 16);
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n"
                   ::"r"(dst + (uint32_t)(at - (first & ~uintptr_t(15)))), "l"(reinterpret_cast<const void*>(at)), "r"(bytes) : "memory");
    }
  }
}
template <typename T>
__device__ __forceinline__ const T* span_at(const char* buffer, const T* row, int begin) {
  return reinterpret_cast<const T*>(buffer + (reinterpret_cast<uintptr_t>(row + begin) & 15));
}

__device__ __forceinline__ uint32_t smem_of(const void* x) { return static_cast<uint32_t>(__cvta_generic_to_shared(x)); }

// The sums of the spans of [begin, end) by one warp, to sums[0 .. count).
template <typename T, bool Q>
__device__ __forceinline__ void sum_spans(const Row<T>& row, int begin, int end, int count, char* ring,
                                          unsigned long long* sums) {
  constexpr int kSpan = kSpanBytes / sizeof(T);
  const int lane = threadIdx.x & 31;
  const uint32_t base = static_cast<uint32_t>(__cvta_generic_to_shared(ring));
  auto issue = [&](int j) {
    const int first = begin + j * kSpan, last = min(end, first + kSpan);
    if (j < count && first < last) {
      copy_span(base + (j % kStages) * 2 * kBuffer, row.p, first, last);
      if (Q) copy_span(base + ((j % kStages) * 2 + 1) * kBuffer, row.q, first, last);
    }
    asm volatile("cp.async.commit_group;\n" ::: "memory");
  };
#pragma unroll
  for (int j = 0; j < kStages - 1; ++j) issue(j);
  for (int j = 0; j < count; ++j) {
    issue(j + kStages - 1);
    asm volatile("cp.async.wait_group %0;\n" ::"n"(kStages - 1) : "memory");
    __syncwarp();
    const int first = begin + j * kSpan, last = min(end, first + kSpan);
    const T* a = span_at(ring + (j % kStages) * 2 * kBuffer, row.p, first);
    const T* b = Q ? span_at(ring + ((j % kStages) * 2 + 1) * kBuffer, row.q, first) : nullptr;
    uint32_t hi = 0u, lo = 0u, n = 0u;
    auto add2 = [&](float2 x, float2 y) {
      add_weights(__saturatef(Q ? x.x - y.x : x.x), __saturatef(Q ? x.y - y.y : x.y), hi, lo);
    };
    if (last - first == kSpan) {
      n = kSpan / 32;
      if constexpr (sizeof(T) == 2) {
        // p's aligned words, two elements each. If the span begins in the middle of one, that word's
        // first element is not the span's: its place is taken by the span's last.
        const int odd = (smem_of(a) >> 1) & 1;
        const T *a2 = a - odd + 2 * lane, *b2 = Q ? b - odd + 2 * lane : nullptr;
        const bool same = Q && (smem_of(b2) & 3) == 0;
        auto words = [&](auto aligned) {
          auto p2 = [&](int e) { return pair_of(*reinterpret_cast<const uint32_t*>(a2 + e * 64), T()); };
          auto q2 = [&](int e) {
            if constexpr (!Q) return make_float2(0.f, 0.f);
            else if constexpr (decltype(aligned)::value) return pair_of(*reinterpret_cast<const uint32_t*>(b2 + e * 64), T());
            else return make_float2(value_of(b2[e * 64]), value_of(b2[e * 64 + 1]));
          };
          float2 x = p2(0), y = q2(0);
          if (odd && lane == 0) {
            x.x = value_of(a[kSpan - 1]);
            if (Q) y.x = value_of(b[kSpan - 1]);
          }
          add2(x, y);
#pragma unroll 5
          for (int e = 1; e < kSpan / 64; ++e) add2(p2(e), q2(e));
        };
        if (same) words(std::true_type());
        else words(std::false_type());
      } else {
#pragma unroll 4
        for (int e = lane; e < kSpan; e += 64)
          add2(make_float2(value_of(a[e]), value_of(a[e + 32])), Q ? make_float2(value_of(b[e]), value_of(b[e + 32])) : make_float2(0.f, 0.f));
      }
    } else {
      for (int e = lane; e < last - first; e += 32, ++n) {
        uint32_t x, y;
        weight_halves(__saturatef(Q ? value_of(a[e]) - value_of(b[e]) : value_of(a[e])), x, y);
        hi += x;
        lo += y;
      }
    }
    unsigned long long s = join(hi, lo, n);
    if (lane == 0 && row.dropped >= first && row.dropped < last) {      // (sums wrap: any lane may take it out)
      uint32_t x, y;
      weight_halves(row.rest(row.dropped), x, y);
      s -= join(x, y, 1);
    }
    s = warp_sum64(s);
    if (lane == 0) __stcg(&sums[j], s);
    __syncwarp();                  // the span is read before its place is filled again
  }
}

// The first element of [begin, end) whose inclusive sum (from `before`) is above the mark, by the
// whole CTA, kScan elements at a time; -1 when there is none.
template <typename T>
__device__ int find_crossing(const Row<T>& row, int begin, int end, unsigned long long before, unsigned long long mark,
                             unsigned long long* sWarp, int* sFound) {
  constexpr int kScan = 1024, kEach = kScan / kThreads;
  for (int v0 = begin; v0 < end; v0 += kScan) {
    const int per = min(kEach, (end - v0 + kThreads - 1) / kThreads);       // consecutive elements of a thread
    unsigned long long mine = 0, total;
#pragma unroll 4
    for (int e = 0; e < kEach; ++e) {
      const int v = v0 + threadIdx.x * per + e;
      mine += e < per && v < end ? row(v) : 0ull;
    }
    const unsigned long long incl = before + block_scan(mine, total, sWarp);
    if (threadIdx.x == 0) *sFound = -1;
    __syncthreads();
    if (incl > mark && incl - mine <= mark) {                // exactly one thread: its elements once more
      unsigned long long at = incl - mine;
      int v = v0 + threadIdx.x * per;
      for (;; ++v) {
        at += row(v);
        if (at > mark) break;
      }
      *sFound = v;
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

// Span c of a row: a warp's share of `share` consecutive elements is per_warp spans. Those past the
// row's end are empty.
template <typename T>
__device__ __forceinline__ void span_range(const VerifyParams& p, int c, int& begin, int& end) {
  constexpr int kSpan = kSpanBytes / sizeof(T);
  const int w = c / p.per_warp, j = c - w * p.per_warp;
  const int64_t lo = (int64_t)w * p.share + j * kSpan;
  begin = (int)min((int64_t)p.V, lo);
  end = (int)min((int64_t)p.V, lo + kSpan);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) verify_kernel(const __grid_constant__ VerifyParams p) {
  extern __shared__ __align__(16) char sRing[];
  __shared__ unsigned long long sWarp[kWarps];
  __shared__ int sRun, sCount, sLast, sFound, sSpan;
  __shared__ unsigned long long sBefore;
  const int b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T* target = reinterpret_cast<const T*>(p.target) + (int64_t)b * p.st[0];
  const T* draft = p.draft == nullptr ? nullptr : reinterpret_cast<const T*>(p.draft) + (int64_t)b * p.sd[0];
  pdl_wait();
  pdl_launch_dependents();
  if (warp == 0) {       // the accepted run: the first refused draft, 32 at a time
    const int n = min(max(p.counts == nullptr ? p.K : p.counts[b], 0), p.K);
    int run = n;
    for (int i0 = 0; i0 < p.K; i0 += 32) {      // (loads of unused drafts too: they do not wait for the count)
      const int i = i0 + lane;
      bool good = i >= n;
      if (i < p.K) {
        const int x = p.tokens[(int64_t)b * p.K + i];
        const float u = p.uniforms[(int64_t)b * (p.K + 1) + i];
        if (x >= 0 && x < p.V) {
          const float q = draft == nullptr ? 1.f : value(draft, (int64_t)i * p.sd[1] + x);
          good |= u * q < value(target, (int64_t)i * p.st[1] + x);
        }
      }
      const unsigned bad = ~__ballot_sync(0xffffffffu, good);
      if (bad) {
        run = i0 + __ffs(bad) - 1;
        break;
      }
    }
    if (lane == 0) {
      sRun = run;
      sCount = n;
    }
  }
  __syncthreads();
  const int run = sRun, n = sCount;
  Row<T> row;
  row.p = target + (int64_t)run * p.st[1];
  row.q = run < n && draft != nullptr ? draft + (int64_t)run * p.sd[1] : nullptr;
  row.dropped = run < n && draft == nullptr ? p.tokens[(int64_t)b * p.K + run] : -1;

  // ---- the spans, by warps
  unsigned long long* sums = p.sums + (int64_t)b * p.spans;
  {
    const int w = blockIdx.x * kWarps + warp;
    const int begin = (int)min((int64_t)p.V, (int64_t)w * p.share), end = (int)min((int64_t)p.V, (int64_t)(w + 1) * p.share);
    char* ring = sRing + warp * kStages * 2 * kBuffer;
    if (row.q != nullptr) sum_spans<T, true>(row, begin, end, p.per_warp, ring, sums + w * p.per_warp);
    else sum_spans<T, false>(row, begin, end, p.per_warp, ring, sums + w * p.per_warp);
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
    int begin, end;
    span_range<T>(p, sSpan, begin, end);
    token = find_crossing(row, begin, end, sBefore, mark, sWarp, &sFound);
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

// About 9 CTAs of 4 warps an SM, at least one a request: more than are resident at once (6),
// because a refused draft doubles a request's bytes and later CTAs even that out. A warp's share
// is whole spans.
void plan_verify(int B, int V, int elem, VerifyPlan& plan) {
  const int most = device_sm_count() * 9 / B > 1 ? device_sm_count() * 9 / B : 1;
  const int span = kSpanBytes / elem;
  const int64_t steps = ((int64_t)V + span - 1) / span;
  for (int64_t each = (steps + (int64_t)most * kWarps - 1) / ((int64_t)most * kWarps);; ++each) {
    const int64_t warps = (steps + each - 1) / each;
    plan.ctas = (int)((warps + kWarps - 1) / kWarps);
    plan.share = (int)(each * span);
    plan.per_warp = (int)each;
    plan.spans = plan.ctas * kWarps * plan.per_warp;
    if (plan.spans <= kMaxSpans || each >= steps) break;
  }
}

namespace {

template <typename T>
int launch(const VerifyParams& p, cudaStream_t st) {
  static bool ready[64] = {false};       // per device: the attribute is set once
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return MA_ERR_CUDA;
  if (dev < 0 || dev >= 64 || !ready[dev]) {
    if (cudaFuncSetAttribute(verify_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingBytes) != cudaSuccess ||
        cudaFuncSetAttribute(verify_kernel<T>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared) !=
            cudaSuccess)
      return MA_ERR_CUDA;
    if (dev >= 0 && dev < 64) ready[dev] = true;
  }
  return launch_pdl(verify_kernel<T>, dim3(p.ctas, p.B), dim3(kThreads), kRingBytes, st, p) == cudaSuccess ? MA_OK : MA_ERR_CUDA;
}

}  // namespace

int launch_verify_drafts(const VerifyParams& p, int dtype, cudaStream_t st) {
  if (dtype == MA_F32) return launch<float>(p, st);
  return dtype == MA_BF16 ? launch<__nv_bfloat16>(p, st) : launch<__half>(p, st);
}

}  // namespace ma
