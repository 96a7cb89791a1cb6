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
// Bound: HBM (160 B per slot and KV head at D = 128) while the rows fit one 8-column MMA tile, the
// products' latency beyond (two warps a scheduler hold the running rows). The rows are the N side (8
// columns) of m16n8k16, the slots (scores) or channels (output) its M side: G = 7 single-token
// rows waste one column of eight, where 128 rows of a tcgen05 tile would waste 121. With the
// slots as a tcgen05 tile's 128 rows instead, every code has to become a 16-bit operand in tensor
// or shared memory first (13 instructions a word of codes against 5 here): that form was built, and
// took 98 us against 60 at 14 rows and 140 against 134 at 35 (32 requests x 8192 slots, 4 KV heads,
// D = 128).
//
// Measured, D = 128, 4 KV heads: 64 requests of 4096 to 16384 slots, 7 rows, 89 us (421 MB: 4.7 TB/s, 73%
// of a copy's rate); 32 such requests, 35 rows, 168 us; 1 request, 8192 slots, 10.7 us, of which the
// chain lengths -> page table -> tiles -> merge takes all but a microsecond or two.
//
// A warp owns 32-slot tiles and a private ring of shared memory filled by cp.async (16-byte
// payload pieces in an XOR swizzle that ldmatrix reads without conflicts, scale and zero
// blocks as they lie), so the main loop has no CTA barrier.
//
// Split: the live slots of all sequences, in units of 256, are cut from the lengths on the device
// (which the host does not know) into whole shares of sequences where those balance, else, as one
// line, into equal ranges that may end one sequence and begin the next; so a ragged batch fills one
// wave of resident CTAs. A sequence cut into several leaves fp32 partials that the last of its CTAs to
// arrive merges in a fixed order. Nobody waits.
#pragma once

#include "ma_kernels.cuh"

namespace ma {

namespace {

constexpr int kTile = kDecodeTile;        // slots per warp tile
constexpr int kUnit = kDecodeUnit;        // granularity of the split in slots
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
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(src) : "memory");
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
__device__ __forceinline__ void ldsm2_t(uint32_t r[2], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0,%1}, [%2];\n" : "=r"(r[0]), "=r"(r[1]) : "r"(addr) : "memory");
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
__device__ __forceinline__ void sts32(uint32_t a, uint32_t v) { asm volatile("st.shared.u32 [%0], %1;\n" ::"r"(a), "r"(v) : "memory"); }
// two fp32 operations in one instruction
__device__ __forceinline__ void add2(float& a0, float& a1, float b0, float b1) {
  asm("{\n.reg .b64 x, y;\nmov.b64 x, {%0, %1};\nmov.b64 y, {%2, %3};\nadd.rn.f32x2 x, x, y;\nmov.b64 {%0, %1}, x;\n}\n"
      : "+f"(a0), "+f"(a1) : "f"(b0), "f"(b1));
}
__device__ __forceinline__ void mul2(float& a0, float& a1, float b0, float b1) {
  asm("{\n.reg .b64 x, y;\nmov.b64 x, {%0, %1};\nmov.b64 y, {%2, %3};\nmul.rn.f32x2 x, x, y;\nmov.b64 {%0, %1}, x;\n}\n"
      : "+f"(a0), "+f"(a1) : "f"(b0), "f"(b1));
}
// (a0, a1) += (c0, c1) * (b0, b1)
__device__ __forceinline__ void fma2(float& a0, float& a1, float c0, float c1, float b0, float b1) {
  asm("{\n.reg .b64 x, y, z;\nmov.b64 x, {%0, %1};\nmov.b64 y, {%2, %3};\nmov.b64 z, {%4, %5};\nfma.rn.f32x2 x, y, z, x;\n"
      "mov.b64 {%0, %1}, x;\n}\n"
      : "+f"(a0), "+f"(a1) : "f"(c0), "f"(c1), "f"(b0), "f"(b1));
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

// 16-byte piece c of slot s's payload row within a stage's payload block: two slots a row of D
// bytes, the pieces of a row XORed with the row so that the pieces of one channel group of
// eight even (or eight odd) slots -- an ldmatrix phase -- lie in different banks.
template <int D>
__device__ __forceinline__ uint32_t piece(int s, int c) {
  const int row = s >> 1, ch = (s & 1) * (D / 32) + c;
  return row * D + ((ch ^ (D == 128 ? row & 7 : (row >> 1) & 3)) << 4);
}

// A CTA's share of one sequence (in shared memory: read where the loops are done).
struct Segment {
  int b;
  int first;      // CTA of the sequence's first share
  int count;      // shares
  int last;       // whether this share ends the sequence
  int begin, end; // its slots
  int next_unit, next_start;    // where the CTA's range goes on, and that sequence's first unit
};

__device__ __forceinline__ int live_slots(const DecodeParams& p, int b) {
  int n = p.kv.nq;
  if (p.kv.lens != nullptr) n = min(n, max(p.kv.lens[b], 0));
  return n;
}
// a sequence without live slots still has a unit: its block keys, or its zero rows
__device__ __forceinline__ int units_of(const DecodeParams& p, int b) {
  return max(1, (live_slots(p, b) + kUnit - 1) / kUnit);
}

// Partial i of a sequence whose first share is in CTA `first`: a CTA has at most two, the share
// that goes on from the CTA before (its even place) and the one that begins a sequence (odd).
__device__ __forceinline__ int partial_slot(int first, int i) { return 2 * (first + i) + (i == 0 ? 1 : 0); }

template <int D>
__device__ __forceinline__ void store_row4(const DecodeParams& p, int b, int h, int r, int d, float4 o) {
  const int g = r / p.T, t = r - g * p.T;
  __nv_bfloat16* dst = p.out + (int64_t)b * p.so[0] + (int64_t)(h * p.G + g) * p.so[1] + (int64_t)t * p.so[2] + d;
  store4(dst, o.x, o.y, o.z, o.w);
}

// A CTA's result from its sources in shared memory -- the block's keys (source 0, unless `skip`) and
// the warps: sRows[1 + W][ROWS][kPad] unnormalized rows, sML[1 + W][ROWS] their (m, l) -- to the
// output rows (normalized) or to partial `slot`. A short sequence leaves most warps without a tile, whose rows
// are not read.
template <int D, int ROWS, int W>
__device__ __forceinline__ void combine(const DecodeParams& p, int b, int h, int r0, int rows, int skip, const float* sRows,
                                        const float2* sML, float2* ml, float* acc) {
  constexpr int kVec = D / 4, kPad = D + 4;
#pragma unroll 1
  for (int i = threadIdx.x; i < rows * kVec; i += W * 32) {
    const int r = i / kVec, d = (i % kVec) * 4;
    float2 e[W + 1];
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w <= W; ++w) {
      e[w] = sML[w * ROWS + r];
      if (w == 0 && skip) e[w] = make_float2(-INFINITY, 0.f);
      m = fmaxf(m, e[w].x);
    }
    const float ms = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w <= W; ++w) {
      const float f = ex2(e[w].x - ms);
      if (f == 0.f) continue;          // (a NaN counts)
      const float4 v = *reinterpret_cast<const float4*>(sRows + (w * ROWS + r) * kPad + d);
      l = fmaf(f, e[w].y, l);
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

// The merge of a sequence's partials, in the last of its CTAs: a few splits at a time come into
// shared memory by one round of cp.async (their latency, not their bytes, is the cost), then
// a thread per four channels of a row folds them. The order is fixed, so the result does not
// depend on who came last. buf: kMerge<...> splits' rows and (m, l).
template <int D, int ROWS, int W>
__device__ __forceinline__ void merge_partials(const DecodeParams& p, const Segment& s, int b, int h, int r0, int rows,
                                               const float2* ml, const float* acc, char* buf, int cap) {
  constexpr int kVec = D / 4, kItems = (ROWS * kVec + W * 32 - 1) / (W * 32);
  const uint32_t dst = smem_u32(buf);
  const uint32_t dst_ml = dst + cap * ROWS * D * 4;
  const float* sAcc = reinterpret_cast<const float*>(buf);
  const float2* sML = reinterpret_cast<const float2*>(buf + cap * ROWS * D * 4);
  float m[kItems], l[kItems];
  float4 o[kItems];
#pragma unroll
  for (int k = 0; k < kItems; ++k) {
    m[k] = -INFINITY;
    l[k] = 0.f;
    o[k] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
#pragma unroll 1
  for (int i0 = 0; i0 < s.count; i0 += cap) {
    const int n = min(cap, s.count - i0);
    __syncthreads();                                  // the rows before are read
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
      const int64_t at = (int64_t)partial_slot(s.first, i0 + i) * ROWS;
#pragma unroll
      for (int k = 0; k < kItems; ++k) {
        const int x = k * W * 32 + threadIdx.x;
        if (x < rows * kVec) cp_async16(dst + (i * ROWS * kVec + x) * 16, acc + at * D + x * 4);
      }
      if (threadIdx.x < ROWS / 2) cp_async16(dst_ml + (i * ROWS + threadIdx.x * 2) * 8, ml + at + threadIdx.x * 2);
    }
    cp_commit();
    cp_wait<0>();
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      const int x = k * W * 32 + threadIdx.x, r = x / kVec;
      if (r >= rows) break;
#pragma unroll 4
      for (int i = 0; i < n; ++i) {
        const float2 e = sML[i * ROWS + r];
        const float4 v = *reinterpret_cast<const float4*>(sAcc + (i * ROWS * kVec + x) * 4);
        const float mn = fmaxf(m[k], e.x), ms = mn == -INFINITY ? 0.f : mn;
        const float f = ex2(m[k] - ms), w = ex2(e.x - ms);
        m[k] = mn;
        l[k] = fmaf(l[k], f, w * e.y);
        o[k].x = fmaf(w, v.x, o[k].x * f);
        o[k].y = fmaf(w, v.y, o[k].y * f);
        o[k].z = fmaf(w, v.z, o[k].z * f);
        o[k].w = fmaf(w, v.w, o[k].w * f);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < kItems; ++k) {
    const int x = k * W * 32 + threadIdx.x, r = x / kVec;
    if (r >= rows) break;
    const float inv = l[k] > 0.f ? 1.f / l[k] : 0.f;
    store_row4<D>(p, b, h, r0 + r, (x % kVec) * 4, make_float4(o[k].x * inv, o[k].y * inv, o[k].z * inv, o[k].w * inv));
  }
}

// The CTA's rows: the output when they are the sequence's only split, else this split's partial
// and, in the last CTA to arrive, the merge of all of them.
template <int D, int ROWS, int W>
__device__ __forceinline__ void finish(const DecodeParams& p, const Segment& s, int h, int rt, int share, int skip,
                                       const float* sRows, const float2* sML, char* buf, int cap) {
  __shared__ int sLast;
  const int r0 = rt * ROWS, rows = min(ROWS, p.R - r0);
  const int b = s.b;
  const int64_t base = (int64_t)(h * p.row_tiles + rt) * 2 * p.ctas * ROWS;
  float2* ml = p.ml + base;
  float* acc = p.acc + base * D;
  const int64_t slot = partial_slot(s.first, share) * (int64_t)ROWS;
  const bool whole = s.count == 1;
  combine<D, ROWS, W>(p, b, h, r0, rows, skip, sRows, sML, ml + slot, whole ? nullptr : acc + slot * D);
  if (whole) return;
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
  merge_partials<D, ROWS, W>(p, s, b, h, r0, rows, ml, acc, buf, cap);
}

// The step's own keys, in fp32 on the CUDA cores: a warp per up to four rows at once (their loads and
// sums overlap: with one at a time a short request waited longer here than for its cache), a lane per
// D/32 channels. Its few keys stay in L1; as bf16 MMA tiles they would need a path of their own.
template <int D, int ROWS, int W>
__device__ void block_rows(const DecodeParams& p, int b, int h, int r0, int rows, float* sRows, float2* sML) {
  constexpr int kPad = D + 4, kCh = D / 32, kR = ROWS / W < 1 ? 1 : ROWS / W > 4 ? 4 : ROWS / W;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const __nv_bfloat16* K = reinterpret_cast<const __nv_bfloat16*>(p.cur.k) + (int64_t)b * p.cur.sk[0] + (int64_t)h * p.cur.sk[1] + lane * kCh;
  const __nv_bfloat16* V = reinterpret_cast<const __nv_bfloat16*>(p.cur.v) + (int64_t)b * p.cur.sv[0] + (int64_t)h * p.cur.sv[1] + lane * kCh;
  auto load = [](const __nv_bfloat16* x, float f[kCh]) {
    if constexpr (kCh == 4) {
      const uint2 u = *reinterpret_cast<const uint2*>(x);
      const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.x));
      const float2 c = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.y));
      f[0] = a.x; f[1] = a.y; f[2] = c.x; f[3] = c.y;
    } else {
      const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(x));
      f[0] = a.x; f[1] = a.y;
    }
  };
#pragma unroll 1
  for (int first = warp; first < rows; first += W * kR) {
    int seen[kR], most = 0;          // a row sees the block's first `seen` keys
    float q[kR][kCh], o[kR][kCh], m[kR], l[kR];
#pragma unroll
    for (int i = 0; i < kR; ++i) {
      const int r = min(first + W * i, rows - 1);      // (rows past the last: the last once more)
      const int g = (r0 + r) / p.T, t = (r0 + r) - g * p.T;
      seen[i] = p.causal ? min(p.cur.Tc, t + p.cur.Tc - p.T + 1) : p.cur.Tc;
      most = max(most, seen[i]);
      load(p.q + (int64_t)b * p.sq[0] + (int64_t)(h * p.G + g) * p.sq[1] + (int64_t)t * p.sq[2] + lane * kCh, q[i]);
      m[i] = -INFINITY;
      l[i] = 0.f;
#pragma unroll
      for (int c = 0; c < kCh; ++c) o[i][c] = 0.f;
    }
#pragma unroll 1
    for (int j0 = 0; j0 < most; j0 += 32) {
      const int nj = min(32, most - j0);
      float v[kCh], pr[kR];
      load(V + (int64_t)j0 * p.cur.sv[2], v);          // with the first key, not after its score
#pragma unroll
      for (int i = 0; i < kR; ++i) pr[i] = -INFINITY;
#pragma unroll 2
      for (int j = 0; j < nj; ++j) {
        float k[kCh];
        load(K + (int64_t)(j0 + j) * p.cur.sk[2], k);
#pragma unroll
        for (int i = 0; i < kR; ++i) {
          float dot = 0.f;
#pragma unroll
          for (int c = 0; c < kCh; ++c) dot = fmaf(q[i][c], k[c], dot);
          dot = warp_sum(dot);
          if (lane == j && j0 + j < seen[i]) pr[i] = dot * p.scale * kLog2e;
        }
      }
#pragma unroll
      for (int i = 0; i < kR; ++i) {
        const float mn = fmaxf(m[i], warp_max(pr[i]));
        const float ms = mn == -INFINITY ? 0.f : mn;
        const float corr = ex2(m[i] - ms);
        pr[i] = ex2(pr[i] - ms);
        m[i] = mn;
        l[i] = l[i] * corr + warp_sum(pr[i]);
#pragma unroll
        for (int c = 0; c < kCh; ++c) o[i][c] *= corr;
      }
#pragma unroll 1
      for (int j = 0; j < nj; ++j) {
        float next[kCh];
        load(V + (int64_t)min(j0 + j + 1, most - 1) * p.cur.sv[2], next);
#pragma unroll
        for (int i = 0; i < kR; ++i) {
          const float w = __shfl_sync(0xffffffffu, pr[i], j);
          if (j0 + j < seen[i]) {      // what a row does not see is not multiplied: it may be NaN
#pragma unroll
            for (int c = 0; c < kCh; ++c) o[i][c] = fmaf(w, v[c], o[i][c]);
          }
        }
#pragma unroll
        for (int c = 0; c < kCh; ++c) v[c] = next[c];
      }
    }
#pragma unroll
    for (int i = 0; i < kR; ++i) {
      const int r = first + W * i;
      if (r >= rows) break;
#pragma unroll
      for (int c = 0; c < kCh; ++c) sRows[r * kPad + lane * kCh + c] = o[i][c];
      if (lane == 0) sML[r] = make_float2(m[i], l[i]);
    }
  }
}

// The query rows of one 8-column tile as B operands, by one warp: q' = q kchan in fp16, scaled by
// a power of two so that a row's largest magnitude lies in [2^13, 2^14) (11 bits of q', where
// a bf16 cache would round k to 8). Lane (g, t4) holds channels 32 gr + 8 t4 + 0..7 of row g; the
// products pair channels (0, 4), (1, 5), (2, 6), (3, 7) of a word as its masks leave them, the
// odd ones with q' / 16 because a high nibble is worth 16 times a low one.
template <int D>
struct QueryTile {
  uint4 b[D / 32][32];     // [group][lane]
  uint32_t z[32];          // B operand of the zero term
  float f[8];              // per row: score in log2 units = f * (sum of products), f > 0
  uint32_t pad[24];
};

// Its global loads (issued before the first copies, so that their latencies overlap) ...
template <int D>
struct QueryLoad {
  uint4 q[D / 32];
  float4 kc[D / 32][2];
  __device__ __forceinline__ void load(const DecodeParams& p, int b, int h, int row0) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    const int r = row0 + g, rg = r / p.T, rt = r - rg * p.T;
    const __nv_bfloat16* x = p.q + (int64_t)b * p.sq[0] + (int64_t)(h * p.G + rg) * p.sq[1] + (int64_t)rt * p.sq[2] + 8 * t4;
    const float* c = p.kv.kchan + (int64_t)b * p.kv.skc[0] + (int64_t)h * p.kv.skc[1] + 8 * t4;
#pragma unroll
    for (int gr = 0; gr < D / 32; ++gr) {
      q[gr] = r < p.R ? *reinterpret_cast<const uint4*>(x + 32 * gr) : make_uint4(0u, 0u, 0u, 0u);
      if (p.kchan_vec) {
        kc[gr][0] = *reinterpret_cast<const float4*>(c + 32 * gr);
        kc[gr][1] = *reinterpret_cast<const float4*>(c + 32 * gr + 4);
      } else {
        const float* e = c + 32 * gr;
        kc[gr][0] = make_float4(e[0], e[1], e[2], e[3]);
        kc[gr][1] = make_float4(e[4], e[5], e[6], e[7]);
      }
    }
  }
};

// ... and what the products take of them.
template <int D>
__device__ __forceinline__ void stage_query(const DecodeParams& p, const QueryLoad<D>& in, QueryTile<D>& out) {
  constexpr int NG = D / 32;
  const int lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  // the scale's sign goes into q', its size into f
  const float sign = p.scale > 0.f ? 1.f : p.scale < 0.f ? -1.f : 0.f, size = p.scale == 0.f ? 1.f : fabsf(p.scale);
  float x[NG][8], amax = 0.f;
#pragma unroll
  for (int gr = 0; gr < NG; ++gr) {
    bf16x8_to_float(in.q[gr], x[gr]);
    const float kc[8] = {in.kc[gr][0].x, in.kc[gr][0].y, in.kc[gr][0].z, in.kc[gr][0].w,
                         in.kc[gr][1].x, in.kc[gr][1].y, in.kc[gr][1].z, in.kc[gr][1].w};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[gr][e] *= kc[e] * sign;
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
    out.b[gr][lane] = make_uint4(pack_half2(x[gr][0], x[gr][4]), pack_half2(x[gr][1] * 0.0625f, x[gr][5] * 0.0625f),
                                 pack_half2(x[gr][2], x[gr][6]), pack_half2(x[gr][3] * 0.0625f, x[gr][7] * 0.0625f));
    z += __shfl_xor_sync(0xffffffffu, z, 1);
    z += __shfl_xor_sync(0xffffffffu, z, 2);
    zg[gr] = z * 0.03125f;       // below 2^14
  }
  // the groups' sums of q' for the zero term, as fp16 high and low parts: together good to 2^-21 of a sum
  // or 2^-20 of the unit of q', so that a group of small q' keeps its part of a score when its zeros are
  // large. (In the codes' unit, 2^-24, the low parts were subnormal: with q' 100 times smaller in the
  // groups whose keys are 100 times larger, and the other way round, outputs were off by 3 %.)
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
  out.z[lane] = low ? pack_half2(z0 - h0, z1 - h1) : pack_half2(h0, h1);
  if (t4 == 0) out.f[g] = size * kLog2e * 16777216.f * __uint_as_float((uint32_t)(eb - 13) << 23);
}

// Shared memory: the query tiles, (m, l) and rows of the results -- the block's first, the warps'
// over the rings, which begin behind the block's.
template <int D, int NT, int W>
__host__ __device__ constexpr uint32_t ring_offset() {
  const size_t before = NT * sizeof(QueryTile<D>) + (size_t)(W + 1) * 8 * NT * 8 + (size_t)8 * NT * (D + 4) * 4;
  return (uint32_t)((before + 127) / 128 * 128);
}

template <int D, int NT, int W>
__host__ __device__ constexpr size_t decode_smem() {
  const size_t ring = ring_offset<D, NT, W>() + (size_t)W * Ring<D>::kWarpBytes;
  const size_t rows = NT * sizeof(QueryTile<D>) + (size_t)(W + 1) * 8 * NT * ((D + 4) * 4 + 8);
  return ring > rows ? ring : rows;
}

// FAST: tiles are contiguous in storage (launch() says when); else every slot is looked up alone.
template <int D, int NT, int W, int MINB, bool FAST>
__global__ void __launch_bounds__(W * 32, MINB) decode_attention_kernel(const __grid_constant__ DecodeParams p) {
  constexpr int ROWS = 8 * NT, NG = D / 32, kPad = D + 4, kSc = D / 16;
  using R = Ring<D>;
  extern __shared__ __align__(128) char smem[];
  __shared__ Segment seg;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t4 = lane & 3;
  const int h = blockIdx.y / p.row_tiles, rt = blockIdx.y - h * p.row_tiles;
  const ma_kv& kv = p.kv;
  QueryTile<D>* query = reinterpret_cast<QueryTile<D>*>(smem);
  const uint32_t ring = smem_u32(smem) + ring_offset<D, NT, W>() + warp * R::kWarpBytes;
  // the result rows of the warps and (the first of them) of the block's keys: the block's have a
  // place of their own before the rings, the warps' lie over them
  float2* sML = reinterpret_cast<float2*>(smem + NT * sizeof(QueryTile<D>));        // [1 + W][ROWS]
  float* sRows = reinterpret_cast<float*>(smem + NT * sizeof(QueryTile<D>) + (W + 1) * ROWS * 8);   // [1 + W][ROWS][kPad]

  pdl_wait();
  pdl_launch_dependents();

  // ---- this CTA's work. Whole shares: every sequence cut into shares of `per` units, one to a CTA,
  // when that takes few more units a CTA than equal ranges would (entering a sequence costs about
  // as much as kEnter units: its query rows, the first copies, its result); else equal ranges. us with kEnter
  // 1 / 2 / 4, one token, D = 128: 20 requests of up to 16384 slots 32.9 / 31.8 / 31.6, 64 of 2048 29.7 / 30.0 / 32.6,
  // 30 of 500 to 9000, 8 heads 50.4 / 50.4 / 53.0.
  constexpr int kEnter = 2, kLeast = 2;
  const int mine0 = lane < p.B ? units_of(p, lane) : 0;        // the first 32 sequences' units, loaded once
  auto units_at = [&](int b) { return b < 32 ? mine0 : units_of(p, b); };     // of this lane's b (b % 32 = lane)
  int all = mine0;
#pragma unroll 1
  for (int b = lane + 32; b < p.B; b += 32) all += units_of(p, b);
  all = __reduce_add_sync(0xffffffffu, all);
  const int ctas = min((int)gridDim.x, (all + kLeast - 1) / kLeast), base = all / ctas, extra = all - base * ctas;
  int per = 0;
  if (p.B <= (int)gridDim.x) {
#pragma unroll 1
    for (int x = max(kLeast, base); x <= base + kEnter && per == 0; ++x) {
      int n = (mine0 + x - 1) / x;
#pragma unroll 1
      for (int b = lane + 32; b < p.B; b += 32) n += (units_of(p, b) + x - 1) / x;
      if (__reduce_add_sync(0xffffffffu, n) <= (int)gridDim.x) per = x;
    }
  }
  // equal ranges: CTA x takes base units, the first `extra` CTAs one more
  auto range_at = [&](int x) { return x * base + min(x, extra); };
  auto cta_of = [&](int u) { return u < extra * (base + 1) ? u / (base + 1) : extra + (u - extra * (base + 1)) / base; };
  const int stop = range_at(blockIdx.x + 1);
  // at: the first unit on the line (ranges) or the CTA's share (whole shares); start: the
  // sequence's first unit or its first CTA
  auto set_segment = [&](int b, int at, int start) {          // by one thread
    const int n = live_slots(p, b), units = max(1, (n + kUnit - 1) / kUnit);
    int lo, hi;
    if (per > 0) {
      lo = (at - start) * per;
      hi = min(units, lo + per);
      seg.first = start;
      seg.count = (units + per - 1) / per;
      seg.next_unit = stop;
    } else {
      lo = at - start;
      hi = min(units, stop - start);
      seg.first = cta_of(start);
      seg.count = cta_of(start + units - 1) - seg.first + 1;
      seg.next_unit = start + hi;
      seg.next_start = start + units;
    }
    seg.b = b;
    seg.last = hi == units;
    seg.begin = lo * kUnit;
    seg.end = (int)min((int64_t)n, (int64_t)hi * kUnit);
  };
  {
    if (per == 0 && (int)blockIdx.x >= ctas) return;
    const int at = per > 0 ? (int)blockIdx.x : range_at(blockIdx.x);
    bool found = false;
#pragma unroll 1
    for (int b0 = 0, done = 0; b0 < p.B && !found; b0 += 32) {
      int n = b0 + lane < p.B ? units_at(b0 + lane) : 0;
      if (per > 0) n = (n + per - 1) / per;
      int incl = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      const bool mine = n > 0 && at >= done + incl - n && at < done + incl;      // at most one lane
      if (mine && warp == 0) set_segment(b0 + lane, at, done + incl - n);
      found = __any_sync(0xffffffffu, mine);
      done += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (!found) return;            // whole shares need fewer CTAs than the grid has
  }
  __syncthreads();

  // the zero term's A operand of the 64-channel form: rows 0, 1 the groups' zeros, 4 ones
  const uint32_t zkeep = g < NG ? 0xffffffffu : 0u, zone = g == 4 ? 0x3C003C00u : 0u;
  // this lane's ldmatrix row: matrix mi = lane / 8 covers rows 8 (mi & 1) .. + 7 (slot 2 row + mt) of
  // group 2 gp + mi / 2; (mt, gp) then flips address bits
  const uint32_t lm = piece<D>(2 * ((lane & 7) + ((lane >> 3) & 1) * 8), lane >> 4);
  // this lane's cp.async destinations: piece `lane` of the block's first 512 bytes, and of its
  // second (the swizzle of 128-byte rows alternates between the two)
  constexpr int kPieces = D / 32, kSlots = 32 / kPieces;       // 16-byte pieces per slot, slots per pass
  const uint32_t cp_dst = piece<D>(lane / kPieces, lane % kPieces);
  constexpr uint32_t kFlip = D == 128 ? 64u : 0u;
  constexpr int kScPieces = kTile * kSc / 16, kScLanes = kTile / kScPieces;    // 16-byte pieces per scale block, slots each

#pragma unroll 1
  while (true) {
    const int b = seg.b, end = seg.end;
    const int tiles = end > seg.begin ? (end - seg.begin + kTile - 1) / kTile : 0;
    const int tile0 = seg.begin / kTile;

    // ---- the copies of a tile of 32 slots into a ring stage. `find` looks a tile up (a load from
    // the page table, one tile ahead of its use), `issue` starts its copies and returns its live
    // slots; dead ones are zero-filled, so nothing stored there is ever multiplied.
    struct Place {
      int page, at;      // FAST: of the tile, else of this lane's slot; page -1: dead
    };
    auto find = [&](int i) -> Place {
      Place f = {-1, 0};
      if constexpr (FAST) {
        if (i < tiles) {
          f.page = b;
          f.at = tile0 + i;
          if (kv.pages != nullptr) {
            const int pi = p.tile_div.div(f.at);
            f.at -= pi * p.tiles_per_page;
            f.page = kv.pages[(int64_t)b * kv.spg + pi];
            if ((unsigned)f.page >= (unsigned)kv.num_pages) f.page = -1;
          }
        }
      } else {
        const int j = (tile0 + i) * kTile + lane;
        if (i < tiles && j < end) {
          kv_page(kv, b, j, f.page, f.at);
          if (kv.mask != nullptr && kv.mask[((int64_t)b * p.H + h) * kv.nq + j] == 0) f.page = -1;
        }
      }
      return f;
    };
    const int64_t hq = (int64_t)h * kv.skq[1], hs = (int64_t)h * kv.sks[1];
    auto issue = [&](int i, uint32_t st, Place f) -> unsigned {
      unsigned alive = 0u;
      if constexpr (FAST) {
        if (i < tiles) {
          const int64_t pg = max(f.page, 0);
          const int64_t oq = hq + pg * kv.skq[0] + (int64_t)f.at * (kTile * D / 2) + lane * 16;
          const int64_t os = (hs + pg * kv.sks[0] + (int64_t)f.at * (kTile * NG)) * 2 + (lane % kScPieces) * 16;
          const uint8_t *sk = kv.kq + oq, *sv = kv.vq + oq;
          const char* ss[NG / 2];
#pragma unroll
          for (int it = 0; it < NG / 2; ++it) {
            // D = 128: K scales and zeros by the half warps, then V's; D = 64: a quarter warp each
            const int blk = (it * 32 + lane) / kScPieces;
            ss[it] = reinterpret_cast<const char*>(blk == 0 ? kv.ks : blk == 1 ? kv.kz : blk == 2 ? kv.vs : kv.vz) + os;
          }
          const int cnt = f.page < 0 ? 0 : min(kTile, end - (tile0 + i) * kTile);
          if (cnt == kTile) {
            alive = 0xffffffffu;
#pragma unroll
            for (int it = 0; it < kPieces; ++it) {
              const uint32_t d = st + (cp_dst ^ ((it & 1) ? kFlip : 0u)) + it * 512;
              cp_async16(d, sk + it * 512);
              cp_async16(d + R::kVq, sv + it * 512);
            }
#pragma unroll
            for (int it = 0; it < NG / 2; ++it) cp_async16(st + R::kKs + (it * 32 + lane) * 16, ss[it]);
          } else {
            alive = (1u << cnt) - 1u;
#pragma unroll
            for (int it = 0; it < kPieces; ++it) {
              const uint32_t d = st + (cp_dst ^ ((it & 1) ? kFlip : 0u)) + it * 512;
              const uint32_t bytes = it * kSlots + lane / kPieces < cnt ? 16u : 0u;
              cp_async<16>(d, sk + it * 512, bytes);
              cp_async<16>(d + R::kVq, sv + it * 512, bytes);
            }
            const uint32_t bytes = min(max((cnt - (lane % kScPieces) * kScLanes) * kSc, 0), 16);
#pragma unroll
            for (int it = 0; it < NG / 2; ++it) cp_async<16>(st + R::kKs + (it * 32 + lane) * 16, ss[it], bytes);
          }
        }
      } else {
        const bool live = f.page >= 0;
        alive = __ballot_sync(0xffffffffu, live);
        if (i < tiles) {
          const int64_t pb = live ? f.page : 0, pj = live ? f.at : 0;
          const int64_t okq = hq + pb * kv.skq[0] + pj * kv.skq[2];
          const int64_t ovq = (int64_t)h * kv.svq[1] + pb * kv.svq[0] + pj * kv.svq[2];
          const int64_t oks = hs + pb * kv.sks[0] + pj * kv.sks[2];
          const int64_t ovs = (int64_t)h * kv.svs[1] + pb * kv.svs[0] + pj * kv.svs[2];
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
            const uint32_t d = st + (cp_dst ^ ((it & 1) ? kFlip : 0u)) + it * 512;
            cp_async<16>(d, kv.kq + ok + c * 16, bytes);
            cp_async<16>(d + R::kVq, kv.vq + ov + c * 16, bytes);
          }
        }
      }
      cp_commit();
      return alive;
    };

    QueryLoad<D> ql;
    if (warp < NT) ql.load(p, b, h, rt * ROWS + warp * 8);
    unsigned flight[kStages];        // live slots of the tiles in flight, the next tile's first
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) flight[i] = issue(warp + i * W, ring + i * R::kStage, find(warp + i * W));
    Place next = find(warp + (kStages - 1) * W);

    static_assert(NT <= W, "a warp per query tile");
    if (warp < NT) stage_query<D>(p, ql, query[warp]);
    const bool with_block = p.cur.Tc > 0 && seg.last;       // the sequence's last share has the block's keys
    if (with_block) block_rows<D, ROWS, W>(p, b, h, rt * ROWS, min(ROWS, p.R - rt * ROWS), sRows, sML);   // while the copies run
    __syncthreads();
    uint32_t zb[NT];
    float fr[NT][2];                 // rows 2 t4 and 2 t4 + 1
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      zb[nt] = query[nt].z[lane];
      fr[nt][0] = query[nt].f[2 * t4];
      fr[nt][1] = query[nt].f[2 * t4 + 1];
    }

    // o: the codes' part; z: the zeros' (lanes g and g + 4 of group g with 128 channels, lane g with
    // 64); l: row sums; all relative to 2^-off: p = 2^(score + off). off brings the largest score
    // to kUp when it is set, and moves only when a later one passes that by kSlack, so that most
    // tiles rescale nothing; p stays below 2^(kUp + kSlack) and, in fp16, normal down to 2^-14.
    constexpr float kUp = 8.f, kSlack = 6.f;
    float o[NT][NG][8], z[NT][2], l[NT][2], off[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int c = 0; c < 2; ++c) z[nt][c] = l[nt][c] = off[nt][c] = 0.f;
#pragma unroll
      for (int gr = 0; gr < NG; ++gr)
#pragma unroll
        for (int i = 0; i < 8; ++i) o[nt][gr][i] = 0.f;
    }
    bool first = true;               // no live tile yet: off is not set
    uint32_t power[NG / 2];          // V scales are used times a power of two per group (fp16, two to a word), so that none reaches 2
#pragma unroll
    for (int e = 0; e < NG / 2; ++e) power[e] = 0x3C003C00u;
    auto power_of = [&](int gr) { return (int)(power[gr / 2] >> (16 * (gr & 1) + 10) & 31u) - 15; };
    auto any_power = [&]() {
      uint32_t x = 0u;
#pragma unroll
      for (int e = 0; e < NG / 2; ++e) x |= power[e] ^ 0x3C003C00u;
      return x != 0u;
    };
    uint32_t stage = ring;           // ring stage of tile i
#pragma unroll 1
    for (int i = warp; i < tiles; i += W) {
      {
        const int nx = i + (kStages - 1) * W;
        flight[kStages - 1] = issue(nx, stage == ring ? ring + (kStages - 1) * R::kStage : stage - R::kStage, next);
        next = find(nx + W);
      }
      cp_wait<kStages - 1>();
      __syncwarp();
      const unsigned alive = flight[0];
#pragma unroll
      for (int e = 0; e < kStages - 1; ++e) flight[e] = flight[e + 1];
      const uint32_t st = stage;
      stage = stage == ring + (kStages - 1) * R::kStage ? ring : stage + R::kStage;
      if (alive == 0u) continue;

      // ---- scores of 2 x 16 slots: the even ones (mt = 0) and the odd ones
      float sc[2][NT][4];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        const uint32_t za = st + R::kKz + (2 * g + mt) * kSc + (NG == 4 ? (t4 & 1) * 4 : 0);
        const uint32_t z0 = lds32(za), z1 = lds32(za + 16 * kSc);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          constexpr float kToCodes = 1.9073486e-6f;      // 2^-19: to the codes' unit
          mma8(sc[mt][nt], z0, z1, zb[nt]);
          mul2(sc[mt][nt][0], sc[mt][nt][1], kToCodes, kToCodes);
          mul2(sc[mt][nt][2], sc[mt][nt][3], kToCodes, kToCodes);
        }
      }
#pragma unroll
      for (int gp = 0; gp < NG / 2; ++gp) {
        uint32_t w[2][4];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) ldsm4(w[mt], st + (lm ^ ((mt * NG + gp * 2) << 4)));
        float2 ksc[2][2];            // K scales of both groups: slots 2 g + mt, + 16
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int hb = 0; hb < 2; ++hb) ksc[mt][hb] = half2_floats(lds32(st + R::kKs + (2 * g + 16 * hb + mt) * kSc + gp * 4));
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int gr = gp * 2 + e;
          uint4 qb[NT];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) qb[nt] = query[nt].b[gr][lane];
#pragma unroll
          for (int mt = 0; mt < 2; ++mt) {
            const uint32_t wa = w[mt][2 * e], wb = w[mt][2 * e + 1], xa = wa >> 8, xb = wb >> 8;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              float c[4];
              mma16_set(c, wa & 0x000F000Fu, wb & 0x000F000Fu, wa & 0x00F000F0u, wb & 0x00F000F0u, qb[nt].x, qb[nt].y);
              mma16(c, xa & 0x000F000Fu, xb & 0x000F000Fu, xa & 0x00F000F0u, xb & 0x00F000F0u, qb[nt].z, qb[nt].w);
              const float k0 = e ? ksc[mt][0].y : ksc[mt][0].x, k1 = e ? ksc[mt][1].y : ksc[mt][1].x;
              fma2(sc[mt][nt][0], sc[mt][nt][1], c[0], c[1], k0, k0);
              fma2(sc[mt][nt][2], sc[mt][nt][3], c[2], c[3], k1, k1);
            }
          }
        }
      }
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int hb = 0; hb < 2; ++hb) {
            float x0 = off[nt][0], x1 = off[nt][1];
            fma2(x0, x1, sc[mt][nt][2 * hb], sc[mt][nt][2 * hb + 1], fr[nt][0], fr[nt][1]);
            sc[mt][nt][2 * hb] = x0;
            sc[mt][nt][2 * hb + 1] = x1;
          }
      if (alive != 0xffffffffu) {
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (!(alive >> (2 * g + mt + (e >> 1) * 16) & 1u)) sc[mt][nt][e] = -INFINITY;
      }

      // ---- references and value scales: rarely anything to do
      float top_x = -INFINITY;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) top_x = fmaxf(top_x, fmaxf(sc[0][nt][e], sc[1][nt][e]));
      uint32_t vtop;                  // this lane's slot's value scales: a set bit 14 is a scale of 2 or more
      if constexpr (NG == 4) {
        const uint2 u = lds64(st + R::kVs + lane * kSc);
        vtop = u.x | u.y;
      } else {
        vtop = lds32(st + R::kVs + lane * kSc);
      }
      if (__any_sync(0xffffffffu, top_x > kUp + kSlack) || first) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float corr[2];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float v = fmaxf(fmaxf(sc[0][nt][c], sc[0][nt][c + 2]), fmaxf(sc[1][nt][c], sc[1][nt][c + 2]));
            v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
            v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
            v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
            const float move = (first || v > kUp) && v != -INFINITY ? v - kUp : 0.f;
            off[nt][c] -= move;
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
              sc[mt][nt][c] -= move;
              sc[mt][nt][c + 2] -= move;
            }
            corr[c] = first ? 0.f : ex2(-move);
            z[nt][c] *= corr[c];
            l[nt][c] *= corr[c];
          }
#pragma unroll
          for (int gr = 0; gr < NG; ++gr)
#pragma unroll
            for (int e = 0; e < 8; ++e) o[nt][gr][e] *= corr[e & 1];
        }
      }
      if (__any_sync(0xffffffffu, (vtop & 0x40004000u) != 0u) || any_power() || first) {
        // The scales of a group are brought below 2 (fp16 products p * scale stay finite), and all of them up to
        // it if a sequence begins with scales below 2^-6 (they stay out of fp16's subnormals). Each group has
        // its own power: one of large values must not push another's scales below what fp16 holds (values
        // of 1000 beside 0.001 with one power: 4 % of the latter's output).
        const uint32_t va = st + R::kVs + lane * kSc;
        uint32_t u[NG / 2], reach = first ? 0x40004000u : 0u;
#pragma unroll
        for (int e = 0; e < NG / 2; ++e) {
          u[e] = lds32(va + e * 4);
          reach |= hmul2(u[e], power[e]);
        }
        if (__any_sync(0xffffffffu, (reach & 0x40004000u) != 0u)) {
          int e5[NG], most = 1;                // exponents of the groups' largest scales in the tile
#pragma unroll
          for (int gr = 0; gr < NG; ++gr) {
            const uint32_t x = u[gr / 2] >> (16 * (gr & 1)) & 0x7fffu;
            e5[gr] = min(max((int)(__reduce_max_sync(0xffffffffu, x) >> 10), 1), 30);
            most = max(most, e5[gr]);
          }
          const int up = most < 9 ? 15 - most : 0;
#pragma unroll
          for (int gr = 0; gr < NG; ++gr) {
            const int is = power_of(gr), to = min(first ? up : is, 15 - e5[gr]);
            if (to != is) {
              const float down = __uint_as_float((uint32_t)(127 + to - is) << 23);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 8; ++e) o[nt][gr][e] *= down;
              const uint32_t half = to > -15 ? (uint32_t)(to + 15) << 10 : 0x0200u;
              power[gr / 2] = gr & 1 ? __byte_perm(power[gr / 2], half, 0x5410) : __byte_perm(half, power[gr / 2], 0x7610);
            }
          }
        }
        if (any_power()) {
          __syncwarp();
#pragma unroll
          for (int e = 0; e < NG / 2; ++e) sts32(va + e * 4, hmul2(u[e], power[e]));
          __syncwarp();
        }
      }

      first = false;

      // ---- probabilities, transposed into B operands
      uint32_t pb[2][NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int hb = 0; hb < 2; ++hb)
            pb[mt][nt][hb] = transpose8x8(pack_half2(ex2(sc[mt][nt][2 * hb]), ex2(sc[mt][nt][2 * hb + 1])));

      // ---- zero term and row sums
      if constexpr (NG == 4) {
        // transposed, the zero block gives rows 0 .. 3 the even slots' zeros and rows 4 .. 7 the odd
        // slots': each product has one half that counts. Rows 8 .. 15 are ones.
        uint32_t a[2];
        ldsm2_t(a, st + R::kVz + (lane & 15) * 16);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float c[4], d[4];
          mma16_set(c, a[0], 0x3C003C00u, a[1], 0x3C003C00u, pb[0][nt][0], pb[0][nt][1]);
          mma16_set(d, a[0], 0x3C003C00u, a[1], 0x3C003C00u, pb[1][nt][0], pb[1][nt][1]);
          add2(z[nt][0], z[nt][1], g < 4 ? c[0] : d[0], g < 4 ? c[1] : d[1]);
          add2(l[nt][0], l[nt][1], c[2], c[3]);
          add2(l[nt][0], l[nt][1], d[2], d[3]);
        }
      } else {
        uint32_t a[2][2];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int hb = 0; hb < 2; ++hb) {
            const uint32_t za = st + R::kVz + (4 * t4 + 16 * hb + mt) * kSc + (g & (NG - 1)) * 2;
            a[mt][hb] = (__byte_perm(lds16(za), lds16(za + 2 * kSc), 0x5410) & zkeep) | zone;
          }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float c[4];
          mma16_set(c, a[0][0], 0x3C003C00u, a[0][1], 0x3C003C00u, pb[0][nt][0], pb[0][nt][1]);
          mma16(c, a[1][0], 0x3C003C00u, a[1][1], 0x3C003C00u, pb[1][nt][0], pb[1][nt][1]);
          add2(z[nt][0], z[nt][1], c[0], c[1]);
          add2(l[nt][0], l[nt][1], c[2], c[3]);
        }
      }

      // ---- codes' part of the output. The tile's products are summed from zero and added to the
      // running sum in fp32: the codes are not centred, so a long chain of the tensor core's
      // truncating additions would leave a bias in the difference of the two parts.
#pragma unroll
      for (int gp = 0; gp < NG / 2; ++gp) {
        uint32_t x[2][4];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) ldsm4_t(x[mt], st + R::kVq + (lm ^ ((mt * NG + gp * 2) << 4)));
        uint32_t vsc[2][2][2];       // V scales of both groups in the slot pairs (4 t4 + mt, + 2) of the B operands
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int hb = 0; hb < 2; ++hb) {
            const uint32_t va = st + R::kVs + (4 * t4 + 16 * hb + mt) * kSc + gp * 4;
            const uint32_t u = lds32(va), v = lds32(va + 2 * kSc);
            vsc[mt][hb][0] = __byte_perm(u, v, 0x5410);
            vsc[mt][hb][1] = __byte_perm(u, v, 0x7632);
          }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int gr = gp * 2 + e;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float c0[4], c1[4];
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
              const uint32_t b0 = hmul2(pb[mt][nt][0], vsc[mt][0][e]), b1 = hmul2(pb[mt][nt][1], vsc[mt][1][e]);
              const uint32_t xa = x[mt][2 * e], xb = x[mt][2 * e + 1], ya = xa >> 8, yb = xb >> 8;
              if (mt == 0) {
                mma16_set(c0, xa & 0x000F000Fu, xa & 0x00F000F0u, xb & 0x000F000Fu, xb & 0x00F000F0u, b0, b1);
                mma16_set(c1, ya & 0x000F000Fu, ya & 0x00F000F0u, yb & 0x000F000Fu, yb & 0x00F000F0u, b0, b1);
              } else {
                mma16(c0, xa & 0x000F000Fu, xa & 0x00F000F0u, xb & 0x000F000Fu, xb & 0x00F000F0u, b0, b1);
                mma16(c1, ya & 0x000F000Fu, ya & 0x00F000F0u, yb & 0x000F000Fu, yb & 0x00F000F0u, b0, b1);
              }
            }
            float* oo = o[nt][gr];
            add2(oo[0], oo[1], c0[0], c0[1]);
            add2(oo[2], oo[3], c0[2], c0[3]);
            add2(oo[4], oo[5], c1[0], c1[1]);
            add2(oo[6], oo[7], c1[2], c1[3]);
          }
        }
      }
      __syncwarp();
    }
    cp_wait<0>();
    __syncthreads();

    // ---- the warps' rows to shared memory (over the rings): o = codes' part + zeros' part
    constexpr float kZ = 1.f / 256.f;     // 2^-kUp
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      if constexpr (NG == 4) {
        z[nt][0] += __shfl_xor_sync(0xffffffffu, z[nt][0], 16);
        z[nt][1] += __shfl_xor_sync(0xffffffffu, z[nt][1], 16);
      }
      float* row = sRows + ((1 + warp) * ROWS + nt * 8 + 2 * t4) * kPad;
#pragma unroll
      for (int gr = 0; gr < NG; ++gr) {
        const float za = __shfl_sync(0xffffffffu, z[nt][0], 4 * gr + t4) * kZ;
        const float zc = __shfl_sync(0xffffffffu, z[nt][1], 4 * gr + t4) * kZ;
        const float unit = __uint_as_float((uint32_t)(127 + 24 - (int)kUp - power_of(gr)) << 23);
        const float* oo = o[nt][gr];
        const int d = 32 * gr + 4 * g;
        *reinterpret_cast<float4*>(row + d) =
            make_float4(fmaf(oo[0], unit, za), fmaf(oo[2], unit * 0.0625f, za), fmaf(oo[4], unit, za), fmaf(oo[6], unit * 0.0625f, za));
        *reinterpret_cast<float4*>(row + kPad + d) =
            make_float4(fmaf(oo[1], unit, zc), fmaf(oo[3], unit * 0.0625f, zc), fmaf(oo[5], unit, zc), fmaf(oo[7], unit * 0.0625f, zc));
      }
      if (g == 0) {
        sML[(1 + warp) * ROWS + nt * 8 + 2 * t4] = make_float2(first ? -INFINITY : kUp - off[nt][0], l[nt][0] * kZ);
        sML[(1 + warp) * ROWS + nt * 8 + 2 * t4 + 1] = make_float2(first ? -INFINITY : kUp - off[nt][1], l[nt][1] * kZ);
      }
    }
    __syncthreads();
    const int skip = with_block ? 0 : 1;
    finish<D, ROWS, W>(p, seg, h, rt, (int)blockIdx.x - seg.first, skip, sRows, sML, smem,
                       (int)(decode_smem<D, NT, W>() / (ROWS * (D * 4 + 8))));
    if (seg.next_unit >= stop) return;
    const int nb = seg.b + 1, at = seg.next_unit, start = seg.next_start;
    __syncthreads();                 // the rows lie over the next sequence's rings
    if (threadIdx.x == 0) set_segment(nb, at, start);
    __syncthreads();
  }
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
  return launch_pdl(kernel, dim3(p.ctas, p.H * p.row_tiles), dim3(W * 32), smem, st, p) == cudaSuccess ? MA_OK : MA_ERR_CUDA;
}

}  // namespace

// The variants of one head dimension. Rows per tile (8 NT): the shapes at which each measured
// fastest are with rows_per_tile() in ma_decode.cu. `wide`: 8 warps of up to 255 registers, one
// CTA an SM, for calls of few units, where a tile's latency counts; else 4 warps and as many
// CTAs as fit without spilling the running rows.
template <int D>
int launch_decode_d(const DecodeParams& p, int rows, bool wide, bool fast, cudaStream_t st) {
  if (!fast) {
    if (wide && rows == 8) return launch<D, 1, 8, 1, false>(p, st);
    if (wide) return launch<D, 2, 8, 1, false>(p, st);
    if (rows == 8) return launch<D, 1, 4, 2, false>(p, st);
    if (rows == 16) return launch<D, 2, 4, 2, false>(p, st);
    return launch<D, 4, 4, 2, false>(p, st);
  }
  if (wide) {
    if (rows == 8) return launch<D, 1, 8, 1, true>(p, st);
    return launch<D, 2, 8, 1, true>(p, st);
  }
  if (rows == 8) return launch<D, 1, 4, 3, true>(p, st);
  // 14 rows, 32 x 8192 slots, 4 KV heads: 3 CTAs an SM (168 registers) 39.5 us against 44.4 for 2 at D = 64; at
  // D = 128, where that spills the running rows, 62.4 against 60.0
  if (rows == 16) return launch<D, 2, 4, D == 64 ? 3 : 2, true>(p, st);
  if (rows == 24) return launch<D, 3, 4, 2, true>(p, st);
  return launch<D, 4, 4, 2, true>(p, st);
}

}  // namespace ma
