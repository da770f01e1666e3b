// AdamW (decoupled weight decay, bias-corrected moments) over many tensors in a few launches, with the moments in 32 or in 8 bits.
//
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2,  p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// 8-bit moments: blocks of 256 consecutive values of a tensor share one fp32 scale, a power of two that puts the block's largest value
// into (128, 256]; a value is an e4m3 code (bias 7, subnormals down to 2^-9: 2^17 below the block's largest).  m is stored as it is, v as
// its ROOT (half the exponent range).  Both are rounded STOCHASTICALLY: a step changes v by about one part in 1 / (1 - b2) = 1000, an e4m3
// step is one part in 8..16, so round-to-nearest would leave v where it is for ever; rounding up with the probability of the cut-off part
// keeps the running averages unbiased.  A v that is not zero never becomes zero (its root divides).  bf16 parameters are rounded the same
// way, for the same reason (a step of 1e-4 of the value against a spacing of 2^-8).  The random bits are a 32-bit integer mix of (seed,
// step, tensor, block, place): nothing depends on the launch, so a step is reproducible bit for bit.
// This file is compiled without FMA contraction: the moments that are rounded to codes are then the same on every path.
#include <algorithm>
#include <cmath>
#include <vector>
#include "kernels.h"
#include "finetune.h"
#include "prof.h"

namespace {
constexpr int AD_TENSORS = 48;           // tensors of one launch: their table rides in the kernel's arguments (no upload, capturable)
constexpr int AD_UNROLL = 4;             // blocks of 256 values a wave works on at a time
constexpr int AD_CHUNK = 4 * AD_UNROLL * ADAMW_BLOCK;   // values of a workgroup of four waves

struct AdTensor {
  void* p;
  const void* g;
  void* m;
  void* v;
  float* ms;
  float* vs;
  int64_t n;
  float decay, size, inv_bc2;            // 1 - lr wd, lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
  unsigned key;
};
struct AdArgs {
  AdTensor t[AD_TENSORS];
  unsigned first[AD_TENSORS + 1];        // workgroups before tensor i
  int count;
  float b1, omb1, b2, omb2, eps, gscale;
};
static_assert(sizeof(AdArgs) <= 4096, "kernel arguments");

// the published finaliser of MurmurHash3 (two multiplications, three shifts); the odd constants it is fed with elsewhere are 2^32 / golden
// ratio and multipliers of published integer hashes, any of which would do
__host__ __device__ __forceinline__ unsigned mix32(unsigned x) {
  x ^= x >> 16;
  x *= 0x85EBCA6Bu;
  x ^= x >> 13;
  x *= 0xC2B2AE35u;
  return x ^ (x >> 16);
}

// A step over more than the last-level cache goes past the caches: it leaves nothing there that the next reader finds, and the memory runs
// 9 % faster without it (519 M parameters: 2.79 -> 2.56 ms); a smaller step's parameters are the next forward's to find.
// four values at `at`, of which `left` (1..4) exist
template <bool NT> __device__ __forceinline__ void load(const float* base, int64_t at, int left, float (&v)[4]) {
  const float* p = base + at;
  if (left >= 4) { const f32x4u t = get<NT>(reinterpret_cast<const f32x4u*>(p)); v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w; return; }
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = i < left ? p[i] : 0.f;
}
template <bool NT> __device__ __forceinline__ void load(const bf16_t* base, int64_t at, int left, float (&v)[4]) {
  const unsigned short* p = (const unsigned short*)base + at;
  unsigned short u[4] = {0, 0, 0, 0};
  if (left >= 4) { const u16x4u t = get<NT>(reinterpret_cast<const u16x4u*>(p)); u[0] = t.x; u[1] = t.y; u[2] = t.z; u[3] = t.w; }
  else {
#pragma unroll
    for (int i = 0; i < 4; ++i) if (i < left) u[i] = p[i];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = __uint_as_float((unsigned)u[i] << 16);
}
template <bool NT> __device__ __forceinline__ void store(float* base, int64_t at, int left, const float (&v)[4]) {
  float* p = base + at;
  if (left >= 4) { const f32x4u t = {v[0], v[1], v[2], v[3]}; put<NT>(reinterpret_cast<f32x4u*>(p), t); return; }
#pragma unroll
  for (int i = 0; i < 4; ++i) if (i < left) p[i] = v[i];
}
template <bool NT> __device__ __forceinline__ void store(bf16_t* base, int64_t at, int left, const unsigned short (&u)[4]) {
  unsigned short* p = (unsigned short*)base + at;
  if (left >= 4) { const u16x4u t = {u[0], u[1], u[2], u[3]}; put<NT>(reinterpret_cast<u16x4u*>(p), t); return; }
#pragma unroll
  for (int i = 0; i < 4; ++i) if (i < left) p[i] = u[i];
}
template <bool NT> __device__ __forceinline__ unsigned load_codes(const unsigned char* p, int left) {
  if (left >= 4) return get<NT>(reinterpret_cast<const u32u*>(p));
  unsigned c = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) if (i < left) c |= (unsigned)p[i] << (8 * i);
  return c;
}
template <bool NT> __device__ __forceinline__ void store_codes(unsigned char* p, int left, unsigned c) {
  if (left >= 4) { put<NT>(reinterpret_cast<u32u*>(p), (u32u)c); return; }
#pragma unroll
  for (int i = 0; i < 4; ++i) if (i < left) p[i] = (unsigned char)(c >> (8 * i));
}
__device__ __forceinline__ void decode(unsigned c, float scale, float (&v)[4]) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
  v[0] = lo.x * scale; v[1] = lo.y * scale; v[2] = hi.x * scale; v[3] = hi.y * scale;
}
// the largest of a wave's 64 values of v, as bits; the lane shifts need no LDS
template <int CTRL> __device__ __forceinline__ unsigned max_with(unsigned x) {
  return max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xF, 0xF, false));
}
// (two at a time: a lane shift waits for the instruction before it)
__device__ __forceinline__ void wave_max(unsigned& x, unsigned& y) {
  x = max_with<0x111>(x); y = max_with<0x111>(y); x = max_with<0x112>(x); y = max_with<0x112>(y);      // within a row of 16 lanes
  x = max_with<0x114>(x); y = max_with<0x114>(y); x = max_with<0x118>(x); y = max_with<0x118>(y);
  x = max_with<0x142>(x); y = max_with<0x142>(y); x = max_with<0x143>(x); y = max_with<0x143>(y);      // over the rows
  x = (unsigned)__builtin_amdgcn_readlane((int)x, 63);
  y = (unsigned)__builtin_amdgcn_readlane((int)y, 63);
}
// 2^k that puts `most` (bits of a finite non-negative float) into (128, 256], and 2^-k
__device__ __forceinline__ void block_scale(unsigned most, float& scale, float& inv) {
  int k = (int)(most >> 23) - 127 + ((most & 0x7FFFFFu) != 0u ? 1 : 0) - 8;
  k = min(max(k, -120), 120);
  scale = __uint_as_float((unsigned)(k + 127) << 23);
  inv = __uint_as_float((unsigned)(127 - k) << 23);
}
// Four e4m3 codes.  v_cvt_sr_fp8_f32 adds the upper 20 of its 32 random bits to what is cut off below the three fraction bits (a
// subnormal: below 2^-9) and truncates: up with the probability of the cut-off part.  The first moment takes the 12 low bits of a value's
// random word (centred), the root the 20 high ones.  NaN becomes the code's NaN; an infinity is not given to it.
template <bool ROOT> __device__ __forceinline__ unsigned encode4(const float (&x)[4], float inv, const unsigned (&rnd)[4]) {
  float y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    y[i] = x[i] * inv;
    if (ROOT) y[i] = y[i] > 0.f ? fmaxf(y[i], 0x1p-9f) : y[i];            // no root but zero becomes zero: at least the least code
  }
  int c = 0;
  c = __builtin_amdgcn_cvt_sr_fp8_f32(y[0], (int)(ROOT ? rnd[0] : (rnd[0] << 20) | 0x80000u), c, 0);
  c = __builtin_amdgcn_cvt_sr_fp8_f32(y[1], (int)(ROOT ? rnd[1] : (rnd[1] << 20) | 0x80000u), c, 1);
  c = __builtin_amdgcn_cvt_sr_fp8_f32(y[2], (int)(ROOT ? rnd[2] : (rnd[2] << 20) | 0x80000u), c, 2);
  c = __builtin_amdgcn_cvt_sr_fp8_f32(y[3], (int)(ROOT ? rnd[3] : (rnd[3] << 20) | 0x80000u), c, 3);
  return (unsigned)c;
}

// One step of four values.  v: the second moment, or its root (8 bits).  The root is correctly rounded - r = x - s^2 is exact in an FMA, so
// one correction of s = x rsq(x) is enough (checked on every fraction) - at half the instructions of sqrtf.  The quotient is a division, as in
// the step over one slab; with 8-bit moments, whose arithmetic is as long as the memory's time, it is m times the hardware's reciprocal, within
// 1.5 ulp, of a change that the moments' 8 bits have made coarser by 2^18.
template <int BITS>
__device__ __forceinline__ void step4(const AdArgs& a, const AdTensor& t, float (&p)[4], const float (&g)[4], float (&m)[4], float (&v)[4],
                                      float (&root)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float gi = g[i] * a.gscale;
    const float vo = BITS == 8 ? v[i] * v[i] : v[i];
    m[i] = m[i] * a.b1 + gi * a.omb1;
    v[i] = vo * a.b2 + (gi * a.omb2) * gi;
    const float y = __builtin_amdgcn_rsqf(v[i]), s = v[i] * y;
    root[i] = fmaf(fmaf(-s, s, v[i]), 0.5f * y, s);
  }
  const float least = fminf(fminf(v[0], v[1]), fminf(v[2], v[3])), most = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
  if (!(least >= 0x1p-90f && most < 0x1p126f)) {                            // zero, next to it, or not finite
#pragma unroll
    for (int i = 0; i < 4; ++i) root[i] = sqrtf(v[i]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float denom = root[i] * t.inv_bc2 + a.eps;
    p[i] = p[i] * t.decay - (BITS == 32 ? m[i] / denom : m[i] * __builtin_amdgcn_rcpf(denom)) * t.size;
  }
}
__device__ __forceinline__ void random4(unsigned key, int64_t blk, int lane, unsigned (&rnd)[4]) {
  const unsigned kb = mix32(key + (unsigned)blk * 0x9E3779B9u);
#pragma unroll
  for (int i = 0; i < 4; ++i) rnd[i] = mix32(kb + (unsigned)(4 * lane + i) * 0x9E3779B9u);
}
__device__ __forceinline__ void round_bf16(const float (&p)[4], const unsigned (&rnd)[4], unsigned short (&w)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned bits = __float_as_uint(p[i]);
    const bool finite = (bits & 0x7FFFFFFFu) < 0x7F800000u;
    w[i] = (unsigned short)((finite ? bits + (mix32(rnd[i] ^ 0x68E31DA4u) & 0xFFFFu) : (p[i] != p[i] ? 0x7FC00000u : bits)) >> 16);
  }
}
// what is left to do of one block when its values are there: `left` (0..4) of the lane's four exist
template <typename PT, int BITS, bool NT>
__device__ __forceinline__ void finish_block(const AdArgs& a, const AdTensor& t, int64_t blk, int lane, int left, float (&p)[4], const float (&g)[4],
                                             float (&m)[4], float (&v)[4]) {
  const int64_t at = blk * ADAMW_BLOCK + 4 * lane;
  unsigned rnd[4] = {0u, 0u, 0u, 0u};
  float root[4];
  if (BITS == 8 || sizeof(PT) == 2) random4(t.key, blk, lane, rnd);
  step4<BITS>(a, t, p, g, m, v, root);
  if (left > 0) {
    if constexpr (sizeof(PT) == 4) store<NT>((float*)t.p, at, left, p);
    else {
      unsigned short w[4];
      round_bf16(p, rnd, w);
      store<NT>((bf16_t*)t.p, at, left, w);
    }
  }
  if constexpr (BITS == 32) {
    if (left > 0) {
      store<NT>((float*)t.m, at, left, m);
      store<NT>((float*)t.v, at, left, v);
    }
  } else {
    unsigned mm = 0u, mv = 0u;                                                // values that do not exist are zeros
#pragma unroll
    for (int i = 0; i < 4; ++i) { mm = max(mm, __float_as_uint(m[i]) & 0x7FFFFFFFu); mv = max(mv, __float_as_uint(root[i]) & 0x7FFFFFFFu); }
    wave_max(mm, mv);
    if (mm >= 0x7F800000u || mv >= 0x7F800000u) {                             // the same in every lane: the scale is that of the finite values, the others are NaN
      mm = mv = 0u;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const unsigned bm = __float_as_uint(m[i]) & 0x7FFFFFFFu, bv = __float_as_uint(root[i]) & 0x7FFFFFFFu;
        if (bm < 0x7F800000u) mm = max(mm, bm); else m[i] = __builtin_nanf("");
        if (bv < 0x7F800000u) mv = max(mv, bv); else root[i] = __builtin_nanf("");
      }
      wave_max(mm, mv);
    }
    float sm, im, sv, iv;
    block_scale(mm, sm, im);
    block_scale(mv, sv, iv);
    const unsigned cm = encode4<false>(m, im, rnd), cv = encode4<true>(root, iv, rnd);
    if (left > 0) {
      store_codes<NT>((unsigned char*)t.m + at, left, cm);
      store_codes<NT>((unsigned char*)t.v + at, left, cv);
    }
    if (lane == 0) { t.ms[blk] = sm; t.vs[blk] = sv; }
  }
}

// A wave takes AD_UNROLL blocks: all their loads are issued before the first is worked on.  A stream: 519 M parameters in 368 tensors, 28
// bytes each with 32-bit moments 2.57 ms = 5.7 TB/s, 16 with 8-bit ones 1.43 ms = 5.8 TB/s (a copy by the library's own kernel reaches 5.5 over
// 4 GiB, 5.7 over 2 and 6.0 over 1); the memory counters see the bytes counted here to 2 %.  The 8-bit form
// stays one as long as its arithmetic is short: with sqrtf, a true division, codes in integer steps and maxima through LDS - 133 vector
// instructions a value - it took 1.90 ms.
template <typename PT, typename GT, int BITS, bool NT>
__global__ void __launch_bounds__(256) adamw_multi_kernel(AdArgs a) {
  // the tensor this workgroup works on
  int lo = 0, hi = a.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.first[mid] <= blockIdx.x) lo = mid; else hi = mid - 1;
  }
  const AdTensor& t = a.t[lo];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t blk0 = ((int64_t)(blockIdx.x - a.first[lo]) * 4 + wave) * AD_UNROLL;
  if ((blk0 + AD_UNROLL) * ADAMW_BLOCK <= t.n) {
    float p[AD_UNROLL][4], g[AD_UNROLL][4], m[AD_UNROLL][4], v[AD_UNROLL][4];
    unsigned cm[AD_UNROLL], cv[AD_UNROLL];
#pragma unroll
    for (int u = 0; u < AD_UNROLL; ++u) {
      const int64_t at = (blk0 + u) * ADAMW_BLOCK + 4 * lane;
      load<NT>((const PT*)t.p, at, 4, p[u]);
      load<NT>((const GT*)t.g, at, 4, g[u]);
      if (BITS == 32) {
        load<NT>((const float*)t.m, at, 4, m[u]);
        load<NT>((const float*)t.v, at, 4, v[u]);
      } else {
        cm[u] = load_codes<NT>((const unsigned char*)t.m + at, 4);
        cv[u] = load_codes<NT>((const unsigned char*)t.v + at, 4);
      }
    }
#pragma unroll
    for (int u = 0; u < AD_UNROLL; ++u) {
      if (BITS == 8) {
        decode(cm[u], t.ms[blk0 + u], m[u]);
        decode(cv[u], t.vs[blk0 + u], v[u]);
      }
      finish_block<PT, BITS, NT>(a, t, blk0 + u, lane, 4, p[u], g[u], m[u], v[u]);
    }
    return;
  }
#pragma unroll 1
  for (int64_t blk = blk0; blk < blk0 + AD_UNROLL && blk * ADAMW_BLOCK < t.n; ++blk) {
    const int64_t at = blk * ADAMW_BLOCK + 4 * lane;
    const int left = at >= t.n ? 0 : (int)min((int64_t)4, t.n - at);
    float p[4] = {0.f, 0.f, 0.f, 0.f}, g[4] = {0.f, 0.f, 0.f, 0.f}, m[4] = {0.f, 0.f, 0.f, 0.f}, v[4] = {0.f, 0.f, 0.f, 0.f};
    if (left > 0) {
      load<NT>((const PT*)t.p, at, left, p);
      load<NT>((const GT*)t.g, at, left, g);
      if (BITS == 32) {
        load<NT>((const float*)t.m, at, left, m);
        load<NT>((const float*)t.v, at, left, v);
      } else {
        decode(load_codes<NT>((const unsigned char*)t.m + at, left), t.ms[blk], m);
        decode(load_codes<NT>((const unsigned char*)t.v + at, left), t.vs[blk], v);
      }
    }
    finish_block<PT, BITS, NT>(a, t, blk, lane, left, p, g, m, v);
  }
}

template <int BITS, bool NT>
int launch_bits(const AdArgs& a, unsigned grid, int pdt, int gdt, hipStream_t s) {
  if (pdt == DT_F32 && gdt == DT_F32) hipLaunchKernelGGL((adamw_multi_kernel<float, float, BITS, NT>), dim3(grid), dim3(256), 0, s, a);
  else if (pdt == DT_F32) hipLaunchKernelGGL((adamw_multi_kernel<float, bf16_t, BITS, NT>), dim3(grid), dim3(256), 0, s, a);
  else if (gdt == DT_F32) hipLaunchKernelGGL((adamw_multi_kernel<bf16_t, float, BITS, NT>), dim3(grid), dim3(256), 0, s, a);
  else hipLaunchKernelGGL((adamw_multi_kernel<bf16_t, bf16_t, BITS, NT>), dim3(grid), dim3(256), 0, s, a);
  HIP_TRY(hipGetLastError());
  return DDMI_OK;
}
}  // namespace

int launch_adamw_multi(const ddmi_adamw_tensor* t, int n, double beta1, double beta2, double eps, double grad_scale, unsigned seed, int pdt, int gdt,
                       int state_bits, hipStream_t s) {
  double values = 0.0;
  for (int i = 0; i < n; ++i) {                // before anything is launched: a call that is refused changes no tensor
    if (cdiv64(t[i].numel, AD_CHUNK) > FT_MOST_GROUPS) return ddmi_fail(DDMI_ERR_INVALID, "adamw_multi: a tensor of more than 2^36 values");
    values += (double)t[i].numel;
  }
  PROF_SCOPE(state_bits == 8 ? "adamw8" : "adamw_multi", 0, values * (2.0 * dt_size(pdt) + dt_size(gdt) + (state_bits == 8 ? 4.0 : 16.0)), s);
  const bool nt = values * (dt_size(pdt) + dt_size(gdt) + (state_bits == 8 ? 2.0 : 8.0)) > FT_CACHE_BYTES;
  AdArgs a;
  a.b1 = (float)beta1; a.omb1 = (float)(1.0 - beta1); a.b2 = (float)beta2; a.omb2 = (float)(1.0 - beta2);
  a.eps = (float)eps; a.gscale = (float)grad_scale;
  int i = 0;
  while (i < n) {
    a.count = 0;
    a.first[0] = 0;
    while (i < n && a.count < AD_TENSORS) {
      const ddmi_adamw_tensor& d = t[i];
      const int64_t wgs = cdiv64(d.numel, AD_CHUNK);
      if (wgs == 0) { ++i; continue; }
      if ((int64_t)a.first[a.count] + wgs > FT_MOST_GROUPS) break;
      AdTensor& o = a.t[a.count];
      o.p = d.param; o.g = d.grad; o.m = d.exp_avg; o.v = d.exp_avg_sq; o.ms = d.exp_avg_scale; o.vs = d.exp_avg_sq_scale; o.n = d.numel;
      o.decay = (float)(1.0 - d.lr * d.weight_decay);
      o.size = (float)(d.lr / (1.0 - std::pow(beta1, (double)d.step)));
      o.inv_bc2 = (float)(1.0 / std::sqrt(1.0 - std::pow(beta2, (double)d.step)));
      o.key = mix32(mix32(mix32(seed) + (unsigned)d.step * 0x9E3779B9u) + (unsigned)(d.index + 1) * 0x85EBCA77u);
      a.first[a.count + 1] = a.first[a.count] + (unsigned)wgs;
      ++a.count;
      ++i;
    }
    if (a.count == 0) continue;
    const unsigned grid = a.first[a.count];
    if (state_bits == 8) DDMI_TRY((nt ? launch_bits<8, true>(a, grid, pdt, gdt, s) : launch_bits<8, false>(a, grid, pdt, gdt, s)));
    else DDMI_TRY((nt ? launch_bits<32, true>(a, grid, pdt, gdt, s) : launch_bits<32, false>(a, grid, pdt, gdt, s)));
  }
  return DDMI_OK;
}
