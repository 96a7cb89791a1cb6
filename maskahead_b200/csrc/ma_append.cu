// New tokens' K/V rows quantized into the slots of a packed (token-mode k4v4) pool: keys and
// values in one launch, through a slot map.
//
// Each row's 32-channel groups are quantized exactly as ma_quantize_tokens does it (the same
// operations rounded to the rows' type in the same order), so a cache filled by prompts in one
// call and by single tokens in many holds the same bytes. A thread has 8 channels: a group's
// minimum and maximum meet in two shuffles, its 16 payload bytes are four neighbouring words,
// and a row of 128 channels is read and written by 16 neighbouring threads.
//
// Bound: HBM (bf16 D = 128: 256 B in, 80 B to the pool, 256 B of values out per row), the launch
// for a few tokens.
#include "ma_kernels.cuh"

namespace ma {

namespace {

constexpr int kGroup = 32;
constexpr int kThreads = 256;

template <bool BF16>
__device__ __forceinline__ float rnd(float x) {
  return BF16 ? __bfloat162float(__float2bfloat16_rn(x)) : x;
}

__device__ __forceinline__ void store8(float* p, const float f[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float f[8]) {
  *reinterpret_cast<uint4*>(p) = float8_to_bf16x8(f);
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) append_kernel(const __grid_constant__ AppendParams p, int64_t rows) {
  constexpr bool BF16 = sizeof(T) == 2;
  constexpr int kLanes = D / 8;                    // threads per row
  const int c = threadIdx.x % kLanes, d = c * 8;
  // rows in the order (token, K or V, head); a warp's rows are a whole number, and every lane
  // stays in the loop for the shuffles
  const int64_t step = (int64_t)gridDim.x * kThreads / kLanes;
  for (int64_t row0 = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / kLanes; __any_sync(0xffffffffu, row0 < rows);
       row0 += step) {
    const bool valid = row0 < rows;
    const int64_t row = valid ? row0 : 0;
    const int h = (int)(row % p.H);
    const int64_t rest = row / p.H;
    const bool key = (rest & 1) == 0;
    const int64_t i = rest >> 1;
    const int seq = p.seqs[i];
    const int64_t slot = p.slots[i];
    const bool owned = seq >= 0 && seq < p.B;
    const T* src = reinterpret_cast<const T*>(key ? p.k : p.v);
    const int64_t* ss = key ? p.sk : p.sv;
    float x[8], kc[8];
    load8(src + i * ss[0] + (int64_t)h * ss[1] + d, x);
    if (key) {
      const float* q = p.kv.kchan + (int64_t)(owned ? seq : 0) * p.kv.skc[0] + (int64_t)h * p.kv.skc[1] + d;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        kc[e] = q[e];
        x[e] = rnd<BF16>(x[e] / kc[e]);
      }
    }
    float mn = x[0], mx = x[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) {
      mn = fminf(mn, x[e]);
      mx = fmaxf(mx, x[e]);
    }
#pragma unroll
    for (int o = 1; o < kGroup / 8; o <<= 1) {
      mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    }
    float s = rnd<BF16>(rnd<BF16>(mx - mn) / 15.0f);
    s = rnd<BF16>(fmaxf(s, 1e-8f));
    uint32_t packed = 0u;
    float back[8];
    const __half sh = __float2half_rn(s), zh = __float2half_rn(mn);
    const float sf = __half2float(sh), zf = __half2float(zh);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float t = rnd<BF16>(rnd<BF16>(x[e] - mn) / s);
      const float code = fminf(fmaxf(rintf(t), 0.f), 15.f);
      packed |= (uint32_t)code << (4 * e);
      back[e] = fmaf(code, sf, zf);
      if (key) back[e] *= kc[e];
    }
    if (!valid) continue;
    T* out = reinterpret_cast<T*>(key ? p.k_rows : p.v_rows);
    if (out != nullptr) {
      if (!owned) {
#pragma unroll
        for (int e = 0; e < 8; ++e) back[e] = 0.f;
      }
      store8(out + (i * p.H + h) * D + d, back);
    }
    if (!owned || slot < 0 || slot >= (int64_t)p.kv.num_pages * p.kv.page_size) continue;
    int64_t page, at;
    if (slot <= 0x7fffffffLL) {
      page = (uint32_t)slot / (uint32_t)p.kv.page_size;
      at = (uint32_t)slot - (uint32_t)page * (uint32_t)p.kv.page_size;
    } else {
      page = slot / p.kv.page_size;
      at = slot - page * p.kv.page_size;
    }
    const int64_t* sq = key ? p.kv.skq : p.kv.svq;
    const int64_t* sc = key ? p.kv.sks : p.kv.svs;
    uint8_t* pay = const_cast<uint8_t*>(key ? p.kv.kq : p.kv.vq);
    *reinterpret_cast<uint32_t*>(pay + page * sq[0] + (int64_t)h * sq[1] + at * sq[2] + c * 4) = packed;
    if ((c & 3) == 0) {
      const int64_t o = page * sc[0] + (int64_t)h * sc[1] + at * sc[2] + c / 4;
      const_cast<uint16_t*>(key ? p.kv.ks : p.kv.vs)[o] = __half_as_ushort(sh);
      const_cast<uint16_t*>(key ? p.kv.kz : p.kv.vz)[o] = __half_as_ushort(zh);
    }
  }
}

template <typename T, int D>
int launch(const AppendParams& p, cudaStream_t st) {
  const int64_t rows = (int64_t)p.N * 2 * p.H;
  const int64_t per = kThreads / (D / 8);
  int64_t grid = (rows + per - 1) / per;
  const int64_t cap = (int64_t)device_sm_count() * 32;
  if (grid > cap) grid = cap;
  append_kernel<T, D><<<(int)grid, kThreads, 0, st>>>(p, rows);
  return cudaGetLastError() == cudaSuccess ? MA_OK : MA_ERR_CUDA;
}

}  // namespace

int launch_append_tokens(const AppendParams& p, int dtype, cudaStream_t st) {
  if (p.N == 0) return MA_OK;
  if (dtype == MA_BF16) return p.D == 128 ? launch<__nv_bfloat16, 128>(p, st) : launch<__nv_bfloat16, 64>(p, st);
  return p.D == 128 ? launch<float, 128>(p, st) : launch<float, 64>(p, st);
}

}  // namespace ma
