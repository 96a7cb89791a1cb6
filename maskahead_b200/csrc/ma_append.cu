// New tokens' K/V rows quantized into the slots of a packed (token-mode k4v4) pool: keys and
// values in one launch, through a slot map.
//
// Each row's 32-channel groups are quantized to the bytes that ma_quantize_tokens gives, so a
// cache filled by prompts in one call and by single tokens in many holds the same. A thread has
// 16 channels, half a group, so that what a row costs beside its elements (its slot, the group's
// minimum and maximum, its step) is shared by many; a row of 128 channels is read and written by
// 8 neighbouring threads. A block takes a run of consecutive tokens, so that a thread keeps its head, its
// channels and, until the request changes, its divisors and their reciprocals.
//
// Bound: HBM (bf16 D = 128: 256 B in, 80 B to the pool, 256 B of values out per row) with the
// issue slots close behind: at the copy's rate an SM has about 26 instructions per element and
// lane. So the bf16 form does without divisions. With 8-bit significands a quotient a / s can
// neither lie on nor within 2^-17 of a boundary of bf16 rounding (m s = a has no solution for a
// 9-bit odd m), so a product with a reciprocal that is off by a few ulps rounds to the same
// bf16. A key's divisor has 24 bits: there the product, 2^-21 of it more and as much less, encloses
// the quotient, and where the two ends round differently (one element in 4000) it is divided.
// 32-bit rows divide keys by their divisors, whose quotients they need to the last bit.
//
// Measured, with values out: 131000 tokens of 4 x 128 in bf16 146 us (622 MB: 4.3 TB/s, 66% of a copy's
// rate; 125 us into consecutive slots, 103 us for a copy of as many bytes), 60000 in 32 bits 110 us (531 MB,
// 4.8 TB/s); 13 tokens 3.2 us, the launch.
#include <type_traits>

#include "ma_kernels.cuh"

namespace ma {

namespace {

constexpr int kThreads = 128;
constexpr int kGroup = 32;
constexpr int kEach = 16;              // channels per thread
constexpr int kPeers = kGroup / kEach; // threads per group

// ---- a thread's channels of one group: x (keys already divided) -> codes, step and minimum
struct Quantized {
  uint32_t packed[kEach / 8];
  __half step, low;
  float code[kEach];
};

// 32-bit rows. A code is the quotient (x - min) / s rounded twice, to 24 bits and to a whole number; the
// product with 1 / s is within 2^-18 of the former (two roundings of 2^-24 of at most 15.1, and the
// quotient's own), so it rounds to the same code unless it lies that close to a half: then (one row
// of 16 in 8000) the quotients are taken.
__device__ __forceinline__ Quantized quantize(const float x[kEach]) {
  float mn = x[0], mx = x[0];
#pragma unroll
  for (int e = 1; e < kEach; ++e) {
    mn = fminf(mn, x[e]);
    mx = fmaxf(mx, x[e]);
  }
#pragma unroll
  for (int o = 1; o < kPeers; o <<= 1) {
    mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  }
  const float s = fmaxf((mx - mn) / 15.0f, 1e-8f);
  Quantized r;
#pragma unroll
  for (int w = 0; w < kEach / 8; ++w) r.packed[w] = 0u;
  const float rs = 1.0f / s;
  bool close = false;
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const float t = (x[e] - mn) * rs, c = rintf(t);
    close |= fabsf(t - c) >= 0.5f - 3.81469727e-6f;
    r.code[e] = fminf(fmaxf(c, 0.f), 15.f);
  }
  if (close) {
#pragma unroll
    for (int e = 0; e < kEach; ++e) r.code[e] = fminf(fmaxf(rintf((x[e] - mn) / s), 0.f), 15.f);
  }
#pragma unroll
  for (int e = 0; e < kEach; ++e) r.packed[e / 8] |= (uint32_t)r.code[e] << (4 * (e & 7));
  r.step = __float2half_rn(s);
  r.low = __float2half_rn(mn);
  return r;
}

__device__ __forceinline__ uint32_t bits(__nv_bfloat162 x) { return *reinterpret_cast<uint32_t*>(&x); }
__device__ __forceinline__ __nv_bfloat162 pair(uint32_t x) { return *reinterpret_cast<__nv_bfloat162*>(&x); }
__device__ __forceinline__ float lo_float(uint32_t x) { return __uint_as_float(x << 16); }
__device__ __forceinline__ float hi_float(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }

// bf16 rows, x in pairs: every operation rounded to bf16, as the quantizer does it.
__device__ __forceinline__ Quantized quantize(const uint32_t x[kEach / 2]) {
  __nv_bfloat162 mn = pair(x[0]), mx = pair(x[0]);
#pragma unroll
  for (int e = 1; e < kEach / 2; ++e) {
    mn = __hmin2(mn, pair(x[e]));
    mx = __hmax2(mx, pair(x[e]));
  }
#pragma unroll
  for (int o = 1; o < kPeers; o <<= 1) {
    mn = __hmin2(mn, pair(__shfl_xor_sync(0xffffffffu, bits(mn), o)));
    mx = __hmax2(mx, pair(__shfl_xor_sync(0xffffffffu, bits(mx), o)));
  }
  const float low = fminf(lo_float(bits(mn)), hi_float(bits(mn))), high = fmaxf(lo_float(bits(mx)), hi_float(bits(mx)));
  const float d = bf16_round(high - low);
  // d / 15 rounds to bf16 as d times the rounded 1/15 does (above)
  const float s = bf16_round(fmaxf(bf16_round(d * (1.0f / 15.0f)), 1e-8f));
  const float rs = __fdividef(1.0f, s);
  const __nv_bfloat162 low2 = __float2bfloat162_rn(low);
  Quantized r;
  uint32_t c[kEach / 2];
  // non-finite rows and steps (s or its reciprocal out of range): the operations as they are
  const bool plain = d < 1e30f;
#pragma unroll
  for (int e = 0; e < kEach / 2; ++e) {
    const uint32_t a = bits(__hsub2(pair(x[e]), low2));
    __nv_bfloat162 t;               // in [0, 15.1] or NaN (-> 0)
    if (plain) {
      t = __hmax2(__floats2bfloat162_rn(lo_float(a) * rs, hi_float(a) * rs), __float2bfloat162_rn(0.f));
    } else {
      t = __hmax2(__floats2bfloat162_rn(lo_float(a) / s, hi_float(a) / s), __float2bfloat162_rn(0.f));
      t = __hmin2(t, __float2bfloat162_rn(15.f));
    }
    // 128 + t rounds t to the nearest whole number, ties to even, and leaves it in the low bits
    const __nv_bfloat162 w = __hadd2(t, __float2bfloat162_rn(128.f));
    const uint32_t code = bits(__hsub2(w, __float2bfloat162_rn(128.f)));
    r.code[2 * e] = lo_float(code);
    r.code[2 * e + 1] = hi_float(code);
    c[e] = bits(w) & 0x000f000fu;
  }
#pragma unroll
  for (int w = 0; w < kEach / 8; ++w) {
    // (c0, c1), (c2, c3) in 16-bit halves -> four nibbles of a half word
    const uint32_t u = c[4 * w] + c[4 * w + 1] * 256u, v = c[4 * w + 2] + c[4 * w + 3] * 256u;
    r.packed[w] = __byte_perm(u | u >> 12, v | v >> 12, 0x5410);
  }
  r.step = __float2half_rn(s);
  r.low = __float2half_rn(low);
  return r;
}

// A thread's divisors and, for bf16 rows, their reciprocals: in shared memory, a column per thread
// (nobody else reads it), which leaves registers for half as many warps again.
template <bool BF16>
struct Divisors {
  static constexpr int kQuads = kEach / 4;
  float4* column;          // [kQuads of kc, kQuads of 1 / kc][kThreads]
  bool usable;
  __device__ __forceinline__ float4 kc(int quad) const { return column[quad * kThreads]; }
  __device__ __forceinline__ float4 r(int quad) const { return column[(kQuads + quad) * kThreads]; }
  __device__ __forceinline__ void load(const float* p) {
    usable = true;
#pragma unroll
    for (int e = 0; e < kQuads; ++e) {
      const float4 k = make_float4(p[4 * e], p[4 * e + 1], p[4 * e + 2], p[4 * e + 3]);
      column[e * kThreads] = k;
      if (BF16) {
        column[(kQuads + e) * kThreads] = make_float4(1.0f / k.x, 1.0f / k.y, 1.0f / k.z, 1.0f / k.w);
        usable &= fminf(fminf(k.x, k.y), fminf(k.z, k.w)) > 1e-30f && fmaxf(fmaxf(k.x, k.y), fmaxf(k.z, k.w)) < 1e30f;
        usable &= k.x == k.x && k.y == k.y && k.z == k.z && k.w == k.w;
      }
    }
  }
};

__device__ __forceinline__ void divide(const Divisors<false>& k, float x[kEach]) {
#pragma unroll
  for (int e = 0; e < kEach / 4; ++e) {
    const float4 d = k.kc(e);
    x[4 * e] /= d.x;
    x[4 * e + 1] /= d.y;
    x[4 * e + 2] /= d.z;
    x[4 * e + 3] /= d.w;
  }
}
constexpr float kAbove = 1.f + 4.76837158e-7f, kBelow = 1.f - 4.76837158e-7f;     // 1 +- 2^-21
__device__ __forceinline__ void divide(const Divisors<true>& k, uint32_t x[kEach / 2]) {
  uint32_t y[kEach / 2], apart = k.usable ? 0u : 1u;
#pragma unroll
  for (int e = 0; e < kEach / 4; ++e) {
    const float4 r = k.r(e);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float a = lo_float(x[2 * e + i]) * (i ? r.z : r.x), b = hi_float(x[2 * e + i]) * (i ? r.w : r.y);
      y[2 * e + i] = bits(__floats2bfloat162_rn(a * kAbove, b * kAbove));
      apart |= y[2 * e + i] ^ bits(__floats2bfloat162_rn(a * kBelow, b * kBelow));
    }
  }
  if (apart) {
#pragma unroll
    for (int e = 0; e < kEach / 4; ++e) {
      const float4 d = k.kc(e);
      y[2 * e] = bits(__floats2bfloat162_rn(lo_float(x[2 * e]) / d.x, hi_float(x[2 * e]) / d.y));
      y[2 * e + 1] = bits(__floats2bfloat162_rn(lo_float(x[2 * e + 1]) / d.z, hi_float(x[2 * e + 1]) / d.w));
    }
  }
#pragma unroll
  for (int e = 0; e < kEach / 2; ++e) x[e] = y[e];
}

__device__ __forceinline__ void load_row(const float* p, float x[kEach]) {
#pragma unroll
  for (int e = 0; e < kEach; e += 4) {
    const float4 u = *reinterpret_cast<const float4*>(p + e);
    x[e] = u.x; x[e + 1] = u.y; x[e + 2] = u.z; x[e + 3] = u.w;
  }
}
__device__ __forceinline__ void load_row(const __nv_bfloat16* p, uint32_t x[kEach / 2]) {
#pragma unroll
  for (int e = 0; e < kEach / 2; e += 4) {
    const uint4 u = *reinterpret_cast<const uint4*>(p + 2 * e);
    x[e] = u.x; x[e + 1] = u.y; x[e + 2] = u.z; x[e + 3] = u.w;
  }
}
__device__ __forceinline__ void store_row(float* p, const float f[kEach]) {
#pragma unroll
  for (int e = 0; e < kEach; e += 4) *reinterpret_cast<float4*>(p + e) = make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
}
__device__ __forceinline__ void store_row(__nv_bfloat16* p, const float f[kEach]) {
#pragma unroll
  for (int e = 0; e < kEach; e += 8) *reinterpret_cast<uint4*>(p + e) = float8_to_bf16x8(f + e);
}

template <typename T, int D, bool KEY>
__device__ __forceinline__ void append_run(const AppendParams& p, int first, int last, int step, int h, int c) {
  using Raw = typename std::conditional<sizeof(T) == 2, uint32_t, float>::type;
  constexpr int kRaw = sizeof(T) == 2 ? kEach / 2 : kEach;
  const T* src = reinterpret_cast<const T*>(KEY ? p.k : p.v) + (int64_t)h * (KEY ? p.sk[1] : p.sv[1]) + c * kEach;
  const int64_t stride = KEY ? p.sk[0] : p.sv[0];
  T* rows = reinterpret_cast<T*>(KEY ? p.k_rows : p.v_rows);
  const int64_t* sq = KEY ? p.kv.skq : p.kv.svq;
  const int64_t* sc = KEY ? p.kv.sks : p.kv.svs;
  uint8_t* pay = const_cast<uint8_t*>(KEY ? p.kv.kq : p.kv.vq) + (int64_t)h * sq[1] + c * (kEach / 2);
  const int64_t sc0 = (int64_t)h * sc[1] + c / kPeers;
  __half* scale = reinterpret_cast<__half*>(const_cast<uint16_t*>(KEY ? p.kv.ks : p.kv.vs)) + sc0;
  __half* zero = reinterpret_cast<__half*>(const_cast<uint16_t*>(KEY ? p.kv.kz : p.kv.vz)) + sc0;
  const int64_t limit = (int64_t)p.kv.num_pages * p.kv.page_size;

  __shared__ float4 sColumns[(KEY ? 2 : 0) * (kEach / 4) + 1][kThreads];
  Divisors<sizeof(T) == 2> kd;
  kd.column = &sColumns[0][threadIdx.x];
  int held = -2;          // the request whose divisors are in kd
  Raw next[kRaw] = {};
  int64_t next_slot = -1;
  int next_seq = -1;
  // pointers to the token that is fetched next, and the row that is written now
  const T* x_at = src + first * stride;
  const int64_t* slot_at = p.slots + first;
  const int32_t* seq_at = p.seqs + first;
  const int64_t x_step = step * stride, row_step = (int64_t)step * p.H * D;
  int64_t row_at = ((int64_t)first * p.H + h) * D + c * kEach;
  auto fetch = [&](int i) {
    if (i < last) {
      load_row(x_at, next);
      next_slot = *slot_at;
      next_seq = *seq_at;
      x_at += x_step;
      slot_at += step;
      seq_at += step;
    }
  };
  fetch(first);
  // the lanes of a row share its token, and every lane of a warp makes the same number of rounds
  const int rounds = __reduce_max_sync(0xffffffffu, (unsigned)(last > first ? (last - first + step - 1) / step : 0));
  for (int k = 0, i = first; k < rounds; ++k, i += step, row_at += row_step) {
    Raw x[kRaw];
#pragma unroll
    for (int e = 0; e < kRaw; ++e) x[e] = next[e];
    const int64_t slot = next_slot;
    const int seq = next_seq;
    const bool valid = i < last, owned = valid && seq >= 0 && seq < p.B;
    fetch(i + step);
    if (KEY) {
      const int want = owned ? seq : 0;
      if (want != held) {
        kd.load(p.kv.kchan + (int64_t)want * p.kv.skc[0] + (int64_t)h * p.kv.skc[1] + c * kEach);
        held = want;
      }
      divide(kd, x);
    }
    const Quantized q = quantize(x);
    if (!valid) continue;
    if (rows != nullptr) {
      const float s = __half2float(q.step), z = __half2float(q.low);
      float back[kEach];
#pragma unroll
      for (int e = 0; e < kEach; ++e) back[e] = fmaf(q.code[e], s, z);
      if (KEY) {
#pragma unroll
        for (int e = 0; e < kEach / 4; ++e) {
          const float4 d = kd.kc(e);
          back[4 * e] *= d.x;
          back[4 * e + 1] *= d.y;
          back[4 * e + 2] *= d.z;
          back[4 * e + 3] *= d.w;
        }
      }
      if (!owned) {
#pragma unroll
        for (int e = 0; e < kEach; ++e) back[e] = 0.f;
      }
      store_row(rows + row_at, back);
    }
    if (!owned || (uint64_t)slot >= (uint64_t)limit) continue;
    uint32_t page, at;                         // (a pool has fewer than 2^31 pages of fewer than 2^31 slots)
    if (slot <= 0x7fffffffLL) page = (uint32_t)p.page_div.div((int)slot);
    else page = (uint32_t)(slot / p.kv.page_size);
    at = (uint32_t)(slot - (int64_t)page * p.kv.page_size);
    *reinterpret_cast<uint2*>(pay + page * (uint64_t)sq[0] + at * (uint64_t)sq[2]) = make_uint2(q.packed[0], q.packed[1]);
    if (c % kPeers == 0) {
      const uint64_t o = page * (uint64_t)sc[0] + at * (uint64_t)sc[2];
      scale[o] = q.step;
      zero[o] = q.low;
    }
  }
}

// grid: (runs of tokens, heads / heads per block, K or V)
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) append_kernel(const __grid_constant__ AppendParams p) {
  constexpr int kLanes = D / kEach;                // threads per row
  const int c = threadIdx.x % kLanes, row = threadIdx.x / kLanes;
  const int sub = row / p.heads_per_block, h = blockIdx.y * p.heads_per_block + row - sub * p.heads_per_block;
  const int step = kThreads / kLanes / p.heads_per_block;
  const int64_t begin = (int64_t)blockIdx.x * p.run;
  const int last = (int)min((int64_t)p.N, begin + p.run);
  const int first = (int)min((int64_t)last, begin + sub);
  pdl_wait();
  pdl_launch_dependents();
  if (blockIdx.z == 0) append_run<T, D, true>(p, first, last, step, h, c);
  else append_run<T, D, false>(p, first, last, step, h, c);
}

template <typename T, int D>
int launch(AppendParams& p, cudaStream_t st) {
  constexpr int kRows = kThreads / (D / kEach);
  p.heads_per_block = kRows % p.H == 0 ? p.H : 1;
  const int step = kRows / p.heads_per_block, groups = p.H / p.heads_per_block;
  // runs of at least one round of the block; at most about 16 blocks an SM over K, V and the heads
  int64_t runs = ((int64_t)p.N + step - 1) / step;
  const int64_t cap = ((int64_t)device_sm_count() * 16 + 2 * groups - 1) / (2 * groups);
  if (runs > cap) runs = cap;
  const int64_t per = ((int64_t)p.N + runs - 1) / runs;
  p.run = (int)((per + step - 1) / step * step);
  runs = ((int64_t)p.N + p.run - 1) / p.run;
  p.page_div.set((uint32_t)p.kv.page_size);
  return launch_pdl(append_kernel<T, D>, dim3((unsigned)runs, groups, 2), dim3(kThreads), 0, st, p) == cudaSuccess ? MA_OK : MA_ERR_CUDA;
}

}  // namespace

int launch_append_tokens(AppendParams& p, int dtype, cudaStream_t st) {
  if (p.N == 0) return MA_OK;
  if (dtype == MA_BF16) return p.D == 128 ? launch<__nv_bfloat16, 128>(p, st) : launch<__nv_bfloat16, 64>(p, st);
  return p.D == 128 ? launch<float, 128>(p, st) : launch<float, 64>(p, st);
}

}  // namespace ma
