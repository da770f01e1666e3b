// Fine-tuning losses of a trained latent diffusion model, each with its gradient: the preference loss (paired log ratios of denoising
// errors against a frozen reference network) and the clipped policy loss with a KL term (log-density of a denoising transition).
//
// Per value, with c = sigmoid(logit[channel]) and m = sqrt(1 - abar_t) x_t (the mixed prediction; without a logit eps = o):
//   eps = m + c (o - m),   eps - eps_ref = c (o - r) + (c - c_ref) (r - m)          (r: the reference's output; no cancellation)
//   preference:  d = eps - noise,                  sums  (eps - eps_ref) (2 d - (eps - eps_ref)) = d^2 - d_ref^2,  d^2,  d (o - m)
//   policy:      z = (x_prev - A x_t) - E eps,     sums  z^2,  (eps - eps_ref)^2,  z (o - m),  (eps - eps_ref) (o - m)
// One scalar (two with KL) a sample follows from the sums over ALL of its values, and only then is the gradient known:
//   d loss / d o = c (k z' + q far).  So: sums_kernel (reads every input once), rows_kernel (a workgroup a pair / transition: the scalar
//   work in 64 bits), grad_kernel (adds up loss and logits' gradients, reads again what the gradient needs and writes it).  A large batch is
//   read once: fused_kernel below.
// Factors are rounded in fp32, products and sums are held in fp64: a margin is the difference of two nearly equal errors times
// beta ~ 10^3, and a logit's gradient a sum of either sign over the batch.  No float atomics: every sum has a fixed order.
#include <algorithm>
#include <atomic>
#include "kernels.h"
#include "finetune.h"
#include "prof.h"

namespace {
// One pass over a large batch leaves nothing in the caches that anyone finds again, and the memory runs faster past them (256 pairs of
// 64 x 64 x 64: 508 -> 473 us; 16 pairs: 62 -> 53)
template <bool NT = false> __device__ __forceinline__ void load4(const float* p, float (&v)[4]) {
  const f32x4u t = get<NT>(reinterpret_cast<const f32x4u*>(p));
  v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
}
__device__ __forceinline__ float bf16_bits(unsigned short u) { return __uint_as_float((unsigned)u << 16); }
template <bool NT = false> __device__ __forceinline__ void load4(const bf16_t* p, float (&v)[4]) {
  const u16x4u t = get<NT>(reinterpret_cast<const u16x4u*>(p));
  v[0] = bf16_bits(t.x); v[1] = bf16_bits(t.y); v[2] = bf16_bits(t.z); v[3] = bf16_bits(t.w);
}
template <bool NT = false> __device__ __forceinline__ void store4(float* p, const float (&v)[4]) {
  const f32x4u t = {v[0], v[1], v[2], v[3]};
  put<NT>(reinterpret_cast<f32x4u*>(p), t);
}
template <bool NT = false> __device__ __forceinline__ void store4(bf16_t* p, const float (&v)[4]) {   // the gradient's one rounding, to the network output's own type
  u16x4u t;
  t.x = __builtin_bit_cast(unsigned short, (bf16_t)v[0]); t.y = __builtin_bit_cast(unsigned short, (bf16_t)v[1]);
  t.z = __builtin_bit_cast(unsigned short, (bf16_t)v[2]); t.w = __builtin_bit_cast(unsigned short, (bf16_t)v[3]);
  put<NT>(reinterpret_cast<u16x4u*>(p), t);
}

// what a workgroup works on: rows [row0, row0 + rows) of sample b, values [t0, t1) of each
struct Span {
  int b, row0, rows, seg;
  int64_t t0, t1;
};
// spans [0, wps) are those of the first sample, and so on; of the preference loss: of the first pair's preferred sample, its rejected one ...
template <int MODE>
__device__ __forceinline__ Span span_of(const FtArgs& a, int blk) {
  Span s;
  const int i = blk / a.wps, j = blk - i * a.wps;
  s.b = MODE == FT_PREF ? (i >> 1) + (i & 1) * a.pairs : i;
  s.row0 = (j / a.nseg) * a.rows_per_wg;
  s.seg = j - (j / a.nseg) * a.nseg;
  s.rows = min(a.rows_per_wg, a.C - s.row0);
  s.t0 = (int64_t)s.seg * a.seg;
  s.t1 = s.t0 + a.seg < a.T ? s.t0 + a.seg : a.T;
  return s;
}
template <int MODE>
__device__ __forceinline__ bool takes_part(const FtArgs& a, int b) {
  if (a.weight && !(a.weight[MODE == FT_PREF ? b % a.pairs : b] > 0.f)) return false;
  // a transition without noise has no density; a deviation that is none (negative, NaN) takes part and shows as NaN: its logarithm is one
  if (MODE == FT_POLICY && a.transition[3 * (int64_t)b + 2] == 0.f) return false;
  return true;
}
// c and c - c_ref of the span's rows; the difference is taken in fp64, it may be far below c
__device__ __forceinline__ void mix_rows(const FtArgs& a, const Span& s, float2* mix) {
  for (int r = threadIdx.x; r < s.rows; r += FT_THREADS) {
    const double c = 1.0 / (1.0 + exp(-(double)a.logit[s.row0 + r]));
    const double cr = a.ref_logit ? 1.0 / (1.0 + exp(-(double)a.ref_logit[s.row0 + r])) : c;
    mix[r] = make_float2((float)c, (float)(c - cr));
  }
  __syncthreads();
}

struct Elem {
  float s1, A, E, c, dc;
};
// the residual whose square is summed, the step away from the reference (before E), and o - m
template <int MODE, bool MIX, bool REF>
__device__ __forceinline__ void element(const Elem& e, float o, float r, float x, float y, float& res, float& far, float& part) {
  const float m = MIX ? e.s1 * x : 0.f;
  part = MIX ? o - m : 0.f;
  const float eps = MIX ? fmaf(e.c, part, m) : o;
  far = REF ? (MIX ? fmaf(e.c, o - r, e.dc * (r - m)) : o - r) : 0.f;
  if (MODE == FT_PREF) res = eps - y;
  else res = fmaf(-e.E, eps, fmaf(-e.A, x, y));
}

template <int MODE, bool MIX, bool REF>
__device__ __forceinline__ void add_up(float res, float far, float part, double& S0, double& S1, double& S2, double& S3) {
  const double r = res, f = far;
  if (MODE == FT_PREF) { S0 = fma(f, 2.0 * r - f, S0); S1 = fma(r, r, S1); }
  else { S0 = fma(r, r, S0); if (REF) S1 = fma(f, f, S1); }
  if (MIX) { S2 = fma(r, (double)part, S2); if (MODE == FT_POLICY && REF) S3 = fma(f, (double)part, S3); }
}

__device__ __forceinline__ double block_sum(double v, double* red) {
  for (int st = 32; st > 0; st >>= 1) v += __shfl_xor(v, st);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  double t = 0.0;
  for (int w = 0; w < FT_THREADS / 64; ++w) t += red[w];
  return t;
}
// sum of the weights of the rows that take part, by one workgroup
template <int MODE>
__device__ __forceinline__ void total_weight(const FtArgs& a, double* red) {
  const int rows = MODE == FT_PREF ? a.pairs : a.B;
  double total = rows;
  if (a.weight || MODE == FT_POLICY) {
    total = 0.0;
    for (int j = threadIdx.x; j < rows; j += FT_THREADS)
      if (takes_part<MODE>(a, j)) total += a.weight ? (double)a.weight[j] : 1.0;
    total = block_sum(total, red);
    __syncthreads();                  // `red` is the caller's again
  }
  if (threadIdx.x == 0) *a.total = total;
}

// Two passes, the first: every input once.  Bound by memory where the batch fills the card (256 pairs of 64 x 64 x 64: 368 us, 5.1 TB/s),
// by the latency of one round of loads where it does not (one pair of 64 x 64: 5 us).
template <int MODE, bool MIX, bool REF, typename T>
__global__ void __launch_bounds__(FT_THREADS) sums_kernel(FtArgs a) {
  __shared__ float2 mix[FT_ROWS];
  __shared__ double red[2][FT_THREADS / 64];
  const int tid = threadIdx.x;
  if (blockIdx.x == 0) total_weight<MODE>(a, red[0]);
  const Span s = span_of<MODE>(a, blockIdx.x);
  const int G = 1 << a.log_g, lane = tid & (G - 1), group = tid >> a.log_g, ngroups = FT_THREADS >> a.log_g;
  const int wpg = G > 64 ? G / 64 : 1;                // waves that share a row
  const bool used = takes_part<MODE>(a, s.b);
  double S0 = 0.0, S1 = 0.0;
  if (MIX && used) mix_rows(a, s, mix);
  Elem e{a.s1 ? a.s1[s.b] : 0.f, 0.f, 1.f, 1.f, 0.f};
  if (MODE == FT_POLICY) { e.A = a.transition[3 * (int64_t)s.b]; e.E = a.transition[3 * (int64_t)s.b + 1]; }
  const int64_t sb = (int64_t)(s.b % a.second_rows) * a.C;
  for (int r0 = 0; r0 < s.rows; r0 += ngroups) {      // uniform trip count: the shuffles below see whole waves
    const int r = r0 + group;
    double S2 = 0.0, S3 = 0.0;
    if (used && r < s.rows) {
      if (MIX) { const float2 c = mix[r]; e.c = c.x; e.dc = c.y; }
      const int64_t base = ((int64_t)s.b * a.C + s.row0 + r) * a.T, base2 = (sb + s.row0 + r) * a.T;
      const T* po = (const T*)a.out + base;
      const T* pr = REF ? (const T*)a.ref + base : nullptr;
      const float* px = (MIX || MODE == FT_POLICY) ? a.x + base : nullptr;
      const float* py = a.second + base2;
      const int64_t nvec = (s.t1 - s.t0) / 4, tail = s.t0 + 4 * nvec;
#pragma unroll 2
      for (int64_t v = lane; v < nvec; v += G) {
        const int64_t t = s.t0 + 4 * v;
        float o[4], q[4] = {0.f, 0.f, 0.f, 0.f}, x[4] = {0.f, 0.f, 0.f, 0.f}, y[4];
        load4(po + t, o);
        if (REF) load4(pr + t, q);
        if (MIX || MODE == FT_POLICY) load4(px + t, x);
        load4(py + t, y);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float res, far, part;
          element<MODE, MIX, REF>(e, o[i], q[i], x[i], y[i], res, far, part);
          add_up<MODE, MIX, REF>(res, far, part, S0, S1, S2, S3);
        }
      }
      if (tail + lane < s.t1) {                        // at most three values, one a lane (a group of fewer lanes takes turns)
        for (int64_t t = tail + lane; t < s.t1; t += G) {
          float res, far, part;
          element<MODE, MIX, REF>(e, to_f32(po[t]), REF ? to_f32(pr[t]) : 0.f, (MIX || MODE == FT_POLICY) ? px[t] : 0.f, py[t], res, far, part);
          add_up<MODE, MIX, REF>(res, far, part, S0, S1, S2, S3);
        }
      }
    }
    if (MIX) {
      const int w = G < 64 ? G : 64;
      for (int st = w >> 1; st > 0; st >>= 1) { S2 += __shfl_xor(S2, st); if (MODE == FT_POLICY && REF) S3 += __shfl_xor(S3, st); }
      if (r < s.rows && (lane & 63) == 0)
        a.chan[(((int64_t)s.b * a.C + s.row0 + r) * a.nseg + s.seg) * wpg + (lane >> 6)] = make_double2(S2, S3);
    }
  }
  for (int st = 32; st > 0; st >>= 1) { S0 += __shfl_xor(S0, st); S1 += __shfl_xor(S1, st); }
  if ((tid & 63) == 0) { red[0][tid >> 6] = S0; red[1][tid >> 6] = S1; }
  __syncthreads();
  if (tid == 0) {
    double t0 = 0.0, t1 = 0.0;
    for (int w = 0; w < FT_THREADS / 64; ++w) { t0 += red[0][w]; t1 += red[1][w]; }
    a.part[blockIdx.x] = make_double2(t0, t1);
  }
}

// the scalar work of one pair / transition, from its sums
struct RowOut {
  double term, stat[3];       // weighted loss; margin, mse, mse | logp, ratio, kl
  float2 coef[2];             // factors of the residual and of the step from the reference: preferred, rejected | transition
};
__device__ __forceinline__ RowOut pref_row(const FtArgs& a, bool used, double w, double2 sw, double2 sl) {
  RowOut o{};
  const double n = (double)a.C * (double)a.T;
  double h = 0.0, dh = 0.0;
  if (used) {
    h = -0.5 * a.beta * (sw.x - sl.x) / n;
    const double t = log1p(exp(-fabs(h))), ls = a.smoothing;              // -log sigma(h) = t - min(h, 0)
    o.term = w * ((1.0 - ls) * (t - fmin(h, 0.0)) + ls * (t + fmax(h, 0.0)));
    dh = w * (ls / (1.0 + exp(-h)) - (1.0 - ls) / (1.0 + exp(h)));
  }
  o.stat[0] = h; o.stat[1] = sw.y / n; o.stat[2] = sl.y / n;
  o.coef[0] = make_float2((float)(-dh * a.beta / n), 0.f);
  o.coef[1] = make_float2((float)(dh * a.beta / n), 0.f);
  return o;
}
__device__ __forceinline__ RowOut policy_row(const FtArgs& a, bool used, double w, int i, double2 s) {
  RowOut o{};
  const double n = (double)a.C * (double)a.T;
  if (!used) return o;
  const double sd = a.transition[3 * (int64_t)i + 2], var = sd * sd, E = a.transition[3 * (int64_t)i + 1];
  o.stat[0] = -s.x / n / (2.0 * var) - log(sd) - 0.91893853320467274178;
  if (!a.logp_old) return o;
  const double adv = a.advantage[i], ratio = exp(o.stat[0] - (double)a.logp_old[i]);
  const double lo = 1.0 - a.clip, hi = 1.0 + a.clip, held = ratio < lo ? lo : (ratio > hi ? hi : ratio);
  const double kl = E * E * s.y / n / (2.0 * var), open = -adv * ratio, bound = -adv * held;
  const bool free = open >= bound, clipped = bound > open;                 // neither: a NaN, which shows in the sum
  o.term = w * ((free ? open : (clipped ? bound : open + bound)) + a.kl_coef * kl);
  o.stat[1] = ratio; o.stat[2] = kl;
  o.coef[0] = make_float2((float)((free ? open * w / (var * n) : (clipped ? 0.0 : open + bound)) * E), (float)(w * a.kl_coef * E * E / (var * n)));
  return o;
}
constexpr unsigned long long FT_OPEN = 0xFFFFFFFFFFFFFFFFull;   // a sum that is not there yet (one pass, below); no sum is stored as this NaN
// the sums of one sample, by one wave: lane i adds those of spans i, i + 64 ...; false when one did not show up within `polls` looks, or
// where another workgroup has waited in vain already (what holds the compute units holds them for all: the whole call waits once)
__device__ __forceinline__ bool wave_sums(const FtArgs& a, int64_t first, int& polls, double2& out) {
  unsigned long long* p = reinterpret_cast<unsigned long long*>(a.part + first);
  double u = 0.0, v = 0.0;
  for (int j0 = 0; j0 < a.wps; j0 += 64) {
    const int j = j0 + (threadIdx.x & 63);
    unsigned long long x = 0, y = 0;
    for (;;) {
      const int late = __hip_atomic_load(a.late, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);      // in flight with the sums
      if (j < a.wps) {
        x = __hip_atomic_load(p + 2 * j, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        y = __hip_atomic_load(p + 2 * j + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
      if (__all(x != FT_OPEN && y != FT_OPEN)) break;
      if (--polls < 0 || __any(late)) return false;
      __builtin_amdgcn_s_sleep(8);
    }
    u += __longlong_as_double((long long)x);
    v += __longlong_as_double((long long)y);
  }
  for (int st = 32; st > 0; st >>= 1) { u += __shfl_xor(u, st); v += __shfl_xor(v, st); }
  out = make_double2(u, v);
  return true;
}
__device__ __forceinline__ double2 sample_sums(const FtArgs& a, int sample, double* red) {
  if (a.fused) {                      // all are there; in the order of the workgroups that waited for them: the same factors to the last bit
    double2 out;
    int polls = 0;
    wave_sums(a, (int64_t)sample * a.wps, polls, out);
    return out;
  }

  double u = 0.0, v = 0.0;
  for (int j = threadIdx.x; j < a.wps; j += FT_THREADS) {
    const double2 p = a.part[(int64_t)sample * a.wps + j];
    u += p.x; v += p.y;
  }
  u = block_sum(u, red);
  v = block_sum(v, red);
  return make_double2(u, v);
}
// one workgroup a pair / transition
template <int MODE>
__global__ void __launch_bounds__(FT_THREADS) rows_kernel(FtArgs a) {
  __shared__ double red[FT_THREADS / 64];
  const int i = blockIdx.x, tid = threadIdx.x;
  const double total = *a.total;
  const bool used = takes_part<MODE>(a, i);
  const double w = used ? (a.weight ? (double)a.weight[i] : 1.0) / total : 0.0;
  RowOut o;
  if (MODE == FT_PREF) {
    const double2 sw = sample_sums(a, 2 * i, red), sl = sample_sums(a, 2 * i + 1, red);
    o = pref_row(a, used, w, sw, sl);
  } else {
    o = policy_row(a, used, w, i, sample_sums(a, i, red));
  }
  if (tid == 0) {
    a.row_out[0][i] = (float)o.stat[0];
    if (MODE == FT_PREF) {
      a.row_out[1][i] = (float)o.stat[1];
      a.row_out[1][i + a.pairs] = (float)o.stat[2];
      a.coef[i] = o.coef[0];
      a.coef[i + a.pairs] = o.coef[1];
    } else if (a.logp_old) {
      a.row_out[1][i] = (float)o.stat[1];
      a.row_out[2][i] = (float)o.stat[2];
      a.coef[i] = o.coef[0];
    }
  }
  if (a.loss && tid == 0) a.term[i] = o.term;
}
// the loss: the rows' terms, in their order
__device__ __forceinline__ void sum_terms(const FtArgs& a, int rows, double* red) {
  double sum = 0.0;
  for (int j = threadIdx.x; j < rows; j += FT_THREADS) sum += a.term[j];
  sum = block_sum(sum, red);
  if (threadIdx.x == 0) *a.loss = (float)sum;
}
__global__ void __launch_bounds__(FT_THREADS) loss_kernel(FtArgs a, int rows) {
  __shared__ double red[FT_THREADS / 64];
  sum_terms(a, rows, red);
}

// ---- one pass: the residuals wait in registers for their sample's sums ----------------------------------------------------------
// A workgroup reads its span, adds up, publishes its two sums, waits for those of the pair's (transition's) other spans and writes the
// gradient from the residuals in its registers: every input is read once.  The sums' own bits are the signal - open_kernel fills their
// places with a NaN that no sum is stored as - so publishing is two relaxed agent-scope stores, with no fence and no counter.  The wait is
// bounded: a workgroup whose neighbours do not show up (other kernels hold the compute units) leaves its span undone, as then do all that
// would have to wait after it, and grad_kernel, which runs after it in any case (loss and logits' gradients need every sample), computes what
// is not done.
std::atomic<int> g_polls{1 << 12};      // some milliseconds; the spans of a row start within microseconds of each other

template <int MODE>
__global__ void __launch_bounds__(FT_THREADS) open_kernel(FtArgs a, int64_t places) {
  __shared__ double red[FT_THREADS / 64];
  unsigned long long* p = reinterpret_cast<unsigned long long*>(a.part);
  for (int64_t i = (int64_t)blockIdx.x * FT_THREADS + threadIdx.x; i < places; i += (int64_t)gridDim.x * FT_THREADS) p[i] = FT_OPEN;
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.late = 0;
  if (blockIdx.x == 0) total_weight<MODE>(a, red);
}
__device__ __forceinline__ void publish(double* place, double v) {
  const unsigned long long bits = v != v ? 0x7FF8000000000000ull : (unsigned long long)__double_as_longlong(v);
  __hip_atomic_store(reinterpret_cast<unsigned long long*>(place), bits, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// four values as they are stored, of which `left` exist: no conversion, so that the next load does not wait for this one
template <typename T> struct Raw;
template <> struct Raw<float> {
  float v[4];
  __device__ __forceinline__ void get(const float* p, int left) {
    if (left == 4) { load4<true>(p, v); return; }
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < left ? p[i] : 0.f;
  }
  __device__ __forceinline__ float at(int i) const { return v[i]; }
};
template <> struct Raw<bf16_t> {
  unsigned v[2];
  __device__ __forceinline__ void get(const bf16_t* q, int left) {
    const unsigned short* p = reinterpret_cast<const unsigned short*>(q);
    if (left == 4) {
      typedef unsigned u32x2u __attribute__((ext_vector_type(2), aligned(2)));
      const u32x2u t = __builtin_nontemporal_load(reinterpret_cast<const u32x2u*>(p));
      v[0] = t.x; v[1] = t.y;
      return;
    }
    v[0] = p[0] | (left > 1 ? (unsigned)p[1] << 16 : 0u);
    v[1] = left > 2 ? p[2] : 0u;
  }
  __device__ __forceinline__ float at(int i) const { return __uint_as_float(i & 1 ? v[i >> 1] & 0xFFFF0000u : v[i >> 1] << 16); }
};
template <typename T> __device__ __forceinline__ void store_some(T* p, int left, const float (&v)[4]) {
  if (left == 4) { store4<true>(p, v); return; }
#pragma unroll
  for (int i = 0; i < 4; ++i) if (i < left) p[i] = from_f32<T>(v[i]);
}

// NV vectors of four values a thread; a row's vectors lie on its G lanes in turn, `turns` to a lane.  Sixteen vectors of residuals (two
// times eight with KL) leave room for four workgroups a compute unit, so that three load while one waits (256 pairs as a graph, 8 | 12 | 16 |
// 20 | 24 vectors: 488 | 506 | 470 | 501 | 509 us; 512 transitions: 605 | 633 | 519 | 520 | 529).  256 pairs of 64 x 64 x 64: 452 us
// for the 2.42 GB that any form has to move, 5.3 TB/s (the memory counters see 2.55: half of the noise that a pair shares is found in the
// caches by its second sample); 512 transitions with KL: 473 us, 5.7 TB/s, 2.70 GB counted of 2.68.  What is left is the wait for the last
// of a sample's spans; loading a vector ahead of its use costs more registers than it gains (2 % slower).
template <int MODE, bool MIX, bool REF, typename T, int NV>
__global__ void __launch_bounds__(FT_THREADS, 2) fused_kernel(FtArgs a) {
  constexpr bool TWO = MODE == FT_POLICY && REF;
  __shared__ float2 mix[FT_ROWS];
  __shared__ double red[2][FT_THREADS / 64];
  __shared__ float2 factor;
  __shared__ int whole;
  const int tid = threadIdx.x;
  const Span s = span_of<MODE>(a, blockIdx.x);
  const int G = 1 << a.log_g, lane = tid & (G - 1), group = tid >> a.log_g, ngroups = FT_THREADS >> a.log_g;
  const int wpg = G > 64 ? G / 64 : 1;
  const int len = (int)(s.t1 - s.t0), turns = cdiv(cdiv(len, 4), G), row_turns = cdiv(s.rows, ngroups);
  const bool used = takes_part<MODE>(a, s.b);
  T* pg = (T*)a.d_out + ((int64_t)s.b * a.C + s.row0) * a.T + s.t0;
  if (!used) {                                                             // its partner's spans still read their places
    if (tid == 0) { publish(&a.part[blockIdx.x].x, 0.0); publish(&a.part[blockIdx.x].y, 0.0); a.done[blockIdx.x] = 1; }
    if (MIX)
      for (int i = tid; i < s.rows * wpg; i += FT_THREADS)
        a.chan[(((int64_t)s.b * a.C + s.row0 + i / wpg) * a.nseg + s.seg) * wpg + i % wpg] = make_double2(0.0, 0.0);
    const float zero[4] = {0.f, 0.f, 0.f, 0.f};
    for (int r = group; r < s.rows; r += ngroups)
      for (int t = 4 * lane; t < len; t += 4 * G) store_some(pg + (int64_t)r * a.T + t, min(4, len - t), zero);
    return;
  }
  if (MIX) mix_rows(a, s, mix);
  Elem e{a.s1 ? a.s1[s.b] : 0.f, 0.f, 1.f, 1.f, 0.f};
  if (MODE == FT_POLICY) { e.A = a.transition[3 * (int64_t)s.b]; e.E = a.transition[3 * (int64_t)s.b + 1]; }
  const int64_t base = ((int64_t)s.b * a.C + s.row0) * a.T + s.t0, base2 = ((int64_t)(s.b % a.second_rows) * a.C + s.row0) * a.T + s.t0;
  const T* po = (const T*)a.out + base;
  const T* pr = REF ? (const T*)a.ref + base : nullptr;
  const float* px = (MIX || MODE == FT_POLICY) ? a.x + base : nullptr;
  const float* py = a.second + base2;
  float res[NV][4], far[TWO ? NV : 1][4];
  double S0 = 0.0, S1 = 0.0, S2 = 0.0, S3 = 0.0;
  int rt = 0, turn = 0;                                                    // the same in every lane
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    if (rt < row_turns) {
      const int r = rt * ngroups + group, t = 4 * (turn * G + lane);
      const int left = r < s.rows ? min(4, len - t) : 0;
      Raw<T> o{}, q{};
      Raw<float> x{}, y{};
      if (left > 0) {
        const int64_t at = (int64_t)r * a.T + t;
        o.get(po + at, left);
        if (REF) q.get(pr + at, left);
        if (MIX || MODE == FT_POLICY) x.get(px + at, left);
        y.get(py + at, left);
        if (MIX) { const float2 c = mix[r]; e.c = c.x; e.dc = c.y; }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float f, part;
          element<MODE, MIX, REF>(e, o.at(i), q.at(i), x.at(i), y.at(i), res[j][i], f, part);
          if (i < left) add_up<MODE, MIX, REF>(res[j][i], f, part, S0, S1, S2, S3);
          if (TWO) far[j][i] = f;
        }
      }
      if (++turn == turns) {                                               // the row is complete
        turn = 0;
        ++rt;
        if (MIX) {
          for (int st = (G < 64 ? G : 64) >> 1; st > 0; st >>= 1) { S2 += __shfl_xor(S2, st); if (TWO) S3 += __shfl_xor(S3, st); }
          if (r < s.rows && (lane & 63) == 0)
            a.chan[(((int64_t)s.b * a.C + s.row0 + r) * a.nseg + s.seg) * wpg + (lane >> 6)] = make_double2(S2, S3);
          S2 = S3 = 0.0;
        }
      }
    }
  }
  for (int st = 32; st > 0; st >>= 1) { S0 += __shfl_xor(S0, st); S1 += __shfl_xor(S1, st); }
  if ((tid & 63) == 0) { red[0][tid >> 6] = S0; red[1][tid >> 6] = S1; }
  __syncthreads();
  if (tid < 64) {
    if (tid == 0) {
      double t0 = 0.0, t1 = 0.0;
      for (int w = 0; w < FT_THREADS / 64; ++w) { t0 += red[0][w]; t1 += red[1][w]; }
      publish(&a.part[blockIdx.x].x, t0);
      publish(&a.part[blockIdx.x].y, t1);
    }
    const int row = MODE == FT_PREF ? s.b % a.pairs : s.b;
    const double w = (a.weight ? (double)a.weight[row] : 1.0) / *a.total;
    int polls = a.polls;
    double2 s0 = make_double2(0.0, 0.0), s1 = make_double2(0.0, 0.0);
    const int64_t first = (int64_t)(MODE == FT_PREF ? 2 * row : row) * a.wps;
    bool ok = wave_sums(a, first, polls, s0);
    if (MODE == FT_PREF && ok) ok = wave_sums(a, first + a.wps, polls, s1);
    const RowOut o = MODE == FT_PREF ? pref_row(a, true, w, s0, s1) : policy_row(a, true, w, row, s0);
    if (tid == 0) {
      const float up = a.dloss ? *a.dloss : 1.f;
      const float2 k = MODE == FT_PREF && s.b >= a.pairs ? o.coef[1] : o.coef[0];
      factor = make_float2(k.x * up, k.y * up);
      whole = ok;
      a.done[blockIdx.x] = ok;
      if (!ok) __hip_atomic_store(a.late, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  __syncthreads();
  if (!whole) return;
  const float2 k = factor;
  rt = turn = 0;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    if (rt < row_turns) {
      const int r = rt * ngroups + group, t = 4 * (turn * G + lane);
      const int left = r < s.rows ? min(4, len - t) : 0;
      if (left > 0) {
        const float c = MIX ? mix[r].x : 1.f, kz = k.x * c, kq = k.y * c;
        float g[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) g[i] = TWO ? fmaf(kq, far[TWO ? j : 0][i], kz * res[j][i]) : kz * res[j][i];
        store_some(pg + (int64_t)r * a.T + t, left, g);
      }
      if (++turn == turns) { turn = 0; ++rt; }
    }
  }
}

// Two passes, the second: the gradient of one span, from the inputs again (387 us for those 256 pairs, 4.9 TB/s).
template <int MODE, bool MIX, bool REF, typename T>
__device__ __forceinline__ void grad_span(const FtArgs& a, int blk, float up, float2* mix) {
  const int tid = threadIdx.x;
  const Span s = span_of<MODE>(a, blk);
  const int G = 1 << a.log_g, lane = tid & (G - 1), group = tid >> a.log_g, ngroups = FT_THREADS >> a.log_g;
  const bool used = takes_part<MODE>(a, s.b);
  if (MIX && used) mix_rows(a, s, mix);
  Elem e{a.s1 ? a.s1[s.b] : 0.f, 0.f, 1.f, 1.f, 0.f};
  if (MODE == FT_POLICY) { e.A = a.transition[3 * (int64_t)s.b]; e.E = a.transition[3 * (int64_t)s.b + 1]; }
  float2 k = a.coef[s.b];
  k.x *= up; k.y *= up;
  const int64_t sb = (int64_t)(s.b % a.second_rows) * a.C;
  for (int r = group; r < s.rows; r += ngroups) {
    if (MIX && used) { const float2 c = mix[r]; e.c = c.x; e.dc = c.y; }
    const float kz = MIX ? k.x * e.c : k.x, kq = MIX ? k.y * e.c : k.y;
    const int64_t base = ((int64_t)s.b * a.C + s.row0 + r) * a.T, base2 = (sb + s.row0 + r) * a.T;
    const T* po = (const T*)a.out + base;
    const T* pr = REF ? (const T*)a.ref + base : nullptr;
    const float* px = (MIX || MODE == FT_POLICY) ? a.x + base : nullptr;
    const float* py = a.second + base2;
    T* pg = (T*)a.d_out + base;
    const int64_t nvec = (s.t1 - s.t0) / 4, tail = s.t0 + 4 * nvec;
#pragma unroll 2
    for (int64_t v = lane; v < nvec; v += G) {
      const int64_t t = s.t0 + 4 * v;
      float g[4] = {0.f, 0.f, 0.f, 0.f};
      if (used) {
        float o[4], q[4] = {0.f, 0.f, 0.f, 0.f}, x[4] = {0.f, 0.f, 0.f, 0.f}, y[4];
        load4(po + t, o);
        if (REF) load4(pr + t, q);
        if (MIX || MODE == FT_POLICY) load4(px + t, x);
        load4(py + t, y);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float res, far, part;
          element<MODE, MIX, REF>(e, o[i], q[i], x[i], y[i], res, far, part);
          g[i] = REF ? fmaf(kq, far, kz * res) : kz * res;
        }
      }
      store4(pg + t, g);
    }
    for (int64_t t = tail + lane; t < s.t1; t += G) {
      float g = 0.f;
      if (used) {
        float res, far, part;
        element<MODE, MIX, REF>(e, to_f32(po[t]), REF ? to_f32(pr[t]) : 0.f, (MIX || MODE == FT_POLICY) ? px[t] : 0.f, py[t], res, far, part);
        g = REF ? fmaf(kq, far, kz * res) : kz * res;
      }
      pg[t] = from_f32<T>(g);
    }
  }
}

// Workgroup 0: the loss; the next `channels`: one channel's logit each; the others take spans in turn, but for those that are in d_out
// already.  `again`: the loss stays, and so does everything where the gradients are those for an upstream gradient of 1 already.
template <int MODE, bool MIX, bool REF, typename T>
__global__ void __launch_bounds__(FT_THREADS) grad_kernel(FtArgs a, int spans, int channels) {
  __shared__ float2 mix[FT_ROWS];
  __shared__ double red[FT_THREADS / 64];
  const int tid = threadIdx.x;
  const float up = a.dloss ? *a.dloss : 1.f;
  const int wg = (int)blockIdx.x - 1 - channels, ch = (int)blockIdx.x - 1;
  if (a.again && up == 1.f) return;
  if (blockIdx.x == 0) {
    if (!a.again) sum_terms(a, MODE == FT_PREF ? a.pairs : a.B, red);
    return;
  }
  if (ch < channels) {
    const int per = a.nseg * (a.log_g > 6 ? 1 << (a.log_g - 6) : 1);
    double s = 0.0;
    for (int64_t j = tid; j < (int64_t)a.B * per; j += FT_THREADS) {
      const int b = (int)(j / per);
      const float2 k = a.coef[b];
      const double2 p = a.chan[((int64_t)b * a.C + ch) * per + (j - (int64_t)b * per)];
      s += k.x * p.x + k.y * p.y;
    }
    s = block_sum(s, red);
    if (tid == 0) {
      const double c = 1.0 / (1.0 + exp(-(double)a.logit[ch]));
      a.d_logit[ch] = (float)(s * c * (1.0 - c) * (double)up);
    }
    return;
  }
  for (int blk = wg; blk < spans; blk += (int)gridDim.x - 1 - channels) {
    if (a.fused && a.done[blk]) continue;
    grad_span<MODE, MIX, REF, T>(a, blk, up, mix);
    __syncthreads();                                    // the next span's coefficients take this one's place
  }
}

template <int MODE, bool MIX, bool REF>
int launch_sums_t(const FtArgs& a, int dt, hipStream_t s) {
  const dim3 grid((unsigned)(a.B * a.wps));
  const int rows = MODE == FT_PREF ? a.pairs : a.B;
  if (a.fused) {
    constexpr int NV = (MODE == FT_POLICY && REF) ? FT_VECS / 2 : FT_VECS;
    const int64_t places = 2ll * a.B * a.wps;
    FtArgs f = a;
    f.polls = g_polls.load(std::memory_order_relaxed);
    hipLaunchKernelGGL((open_kernel<MODE>), dim3((unsigned)std::min<int64_t>(cdiv64(places, FT_THREADS), 256)), dim3(FT_THREADS), 0, s, a, places);
    if (dt == DT_F32) hipLaunchKernelGGL((fused_kernel<MODE, MIX, REF, float, NV>), grid, dim3(FT_THREADS), 0, s, f);
    else hipLaunchKernelGGL((fused_kernel<MODE, MIX, REF, bf16_t, NV>), grid, dim3(FT_THREADS), 0, s, f);
  } else if (dt == DT_F32) {
    hipLaunchKernelGGL((sums_kernel<MODE, MIX, REF, float>), grid, dim3(FT_THREADS), 0, s, a);
  } else {
    hipLaunchKernelGGL((sums_kernel<MODE, MIX, REF, bf16_t>), grid, dim3(FT_THREADS), 0, s, a);
  }
  hipLaunchKernelGGL((rows_kernel<MODE>), dim3((unsigned)rows), dim3(FT_THREADS), 0, s, a);
  if (a.loss && !a.d_out) hipLaunchKernelGGL(loss_kernel, dim3(1), dim3(FT_THREADS), 0, s, a, rows);   // else it is grad_kernel's
  HIP_TRY(hipGetLastError());
  return DDMI_OK;
}
template <int MODE, bool MIX, bool REF>
int launch_grad_t(const FtArgs& a, int dt, hipStream_t s) {
  const int spans = a.B * a.wps, channels = MIX && a.d_logit ? a.C : 0;
  // 1 024 look through what is most often done, 2 048 (eight a compute unit) take what may not have to be done at all
  const dim3 grid((unsigned)(1 + channels + (a.fused ? std::min(spans, 1024) : a.again ? std::min(spans, 2048) : spans)));
  if (dt == DT_F32) hipLaunchKernelGGL((grad_kernel<MODE, MIX, REF, float>), grid, dim3(FT_THREADS), 0, s, a, spans, channels);
  else hipLaunchKernelGGL((grad_kernel<MODE, MIX, REF, bf16_t>), grid, dim3(FT_THREADS), 0, s, a, spans, channels);
  HIP_TRY(hipGetLastError());
  return DDMI_OK;
}
// the gradients times an upstream gradient that is not 1
template <typename T>
__global__ void __launch_bounds__(FT_THREADS) scale_kernel(const float* __restrict__ dloss, T* __restrict__ g, int64_t n, float* __restrict__ d_logit, int C) {
  const float up = *dloss;
  if (up == 1.f) return;
  const int64_t first = (int64_t)blockIdx.x * FT_THREADS + threadIdx.x, step = (int64_t)gridDim.x * FT_THREADS;
  for (int64_t v = first; v < n / 4; v += step) {
    float x[4];
    load4(g + 4 * v, x);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] *= up;
    store4(g + 4 * v, x);
  }
  for (int64_t i = n / 4 * 4 + first; i < n; i += step) g[i] = from_f32<T>(to_f32(g[i]) * up);
  if (d_logit)
    for (int64_t i = first; i < C; i += step) d_logit[i] *= up;
}
}  // namespace

// Two passes: rows are split so that a workgroup has about 8 192 values (16 vectors of four a thread) where there are enough of them for
// 1 024 workgroups, fewer (down to 1 024) where there are not; G lanes share a row, as many as leave each at least two vectors of it, or as there are to share.
// One pass (`keep` vectors a thread stay in registers): a workgroup takes what fills them.
static void ft_split(FtArgs* a, int64_t want) {
  if (a->T > want) {
    a->nseg = (int)std::min<int64_t>(cdiv64(a->T, want), 1 << 20);
    a->seg = cdiv64(cdiv64(a->T, a->nseg), 4) * 4;
    a->nseg = (int)cdiv64(a->T, a->seg);
    a->rows_per_wg = 1;
  } else {
    a->nseg = 1;
    a->seg = cdiv64(a->T, 4) * 4;
    a->rows_per_wg = (int)std::min<int64_t>(std::min<int64_t>(FT_ROWS, a->C), std::max<int64_t>(1, want / a->T));
  }
  a->log_g = 0;
  while (a->log_g < 8 && (((int64_t)16 << a->log_g) <= std::min(a->seg, a->T) || (FT_THREADS >> a->log_g) > a->rows_per_wg)) ++a->log_g;
}
int ft_units() {
  static std::atomic<int> known[64];                    // a device's, plus one; asked once
  int dev = 0, units = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 0;
  if ((units = known[dev].load(std::memory_order_relaxed)) == 0) {
    if (hipDeviceGetAttribute(&units, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess) return 0;
    known[dev].store(++units, std::memory_order_relaxed);
  }
  return units - 1;
}
int ft_plan(FtArgs* a, int B, int C, int64_t HW, bool mixed, int rows_of, int keep, int units) {
  a->B = B;
  a->C = mixed ? C : 1;                       // without a logit nothing depends on the channel: a sample is one row
  a->T = mixed ? HW : HW * C;
  const int64_t all = (int64_t)B * C * HW;
  a->fused = 0;
  if (keep > 0) {
    // whole turns of the groups over the rows, whole turns of the lanes over a row
    ft_split(a, 1024ll * keep);
    const int64_t turns = cdiv64(cdiv64(std::min(a->seg, a->T), 4), 1ll << a->log_g), groups = FT_THREADS >> a->log_g;
    a->rows_per_wg = (int)std::max<int64_t>(1, std::min<int64_t>(a->rows_per_wg, keep / std::max<int64_t>(turns, 1) * groups));
    const int64_t wps = cdiv64(a->C, a->rows_per_wg) * a->nseg;
    // One pass pays from one and a half workgroups a compute unit on, 384 on the whole card's 256 (64 x 64 x 64 latents as graphs, us, two
    // passes | one; 16 workgroups a sample, with KL 32):
    //   samples                 8          12          16          24          32          48         256
    //   preference fp32     30.3|42.9   36.0|44.1   40.9|44.3   49.0|47.1   57.9|51.0   76.3|60.0   407|257
    //   preference bf16     28.0|42.8   34.2|43.6   36.5|43.7   44.7|46.2   48.9|47.0   64.0|51.1   319|201
    //   no mixing fp32      26.1|38.0   29.2|38.4   33.1|39.4   40.8|41.4   45.5|43.5   60.5|50.9   312|208
    //   no mixing bf16      21.6|37.1   26.0|37.5   29.1|38.0   33.3|40.1   37.6|40.9   46.9|43.6   220|151
    //   policy KL fp32      32.2|32.9   39.8|35.1   42.5|36.6   55.0|41.1   63.6|47.5   82.7|65.4   446|259
    //   policy KL bf16      29.7|33.5   35.9|35.1   36.8|35.8   46.1|38.5   51.6|42.3   68.2|58.7   340|221
    //   policy fp32         29.4|39.4   34.9|40.8   37.3|41.7   46.5|43.5   54.2|45.3   68.8|52.6   353|211
    //   policy bf16         27.8|40.0   33.1|40.7   33.9|41.0   41.5|43.1   46.8|43.8   59.2|46.7   288|175
    // One rule for all of them: it is early for bf16 without mixing, whose second reading is the cheapest, by up to 7 us between 384 and 640
    // workgroups, and by 2 us for bf16 with mixing up to 450.  The spans that wait for each other are at most as many as the compute units,
    // each of which holds two: they are resident together with room to spare.  The units are those of the card as it is partitioned.  And the
    // threads' registers are mostly in use.
    const double filled = (double)a->rows_per_wg * (double)std::min(a->seg, a->T) / (1024.0 * keep);
    const bool room = units == FT_ANY_CARD || (units > 0 && 2 * wps * B >= 3 * (int64_t)units && wps * rows_of <= units);
    a->fused = room && turns <= keep && filled >= 0.5;
  }
  if (!a->fused) {
    int64_t want = 8192;
    while (want > 1024 && (double)all / (double)want < 1024.0) want >>= 1;
    ft_split(a, want);
  }
  const int64_t wps = cdiv64(a->C, a->rows_per_wg) * a->nseg;
  if (1 + C + wps * B > FT_MOST_GROUPS) return ddmi_fail(DDMI_ERR_INVALID, "fine-tuning loss: too many values in one call");
  a->wps = (int)wps;
  return DDMI_OK;
}
void ft_set_polls(int n) { g_polls.store(n, std::memory_order_relaxed); }
static size_t up256(size_t b) { return (b + 255) & ~(size_t)255; }
size_t ft_workspace_bytes(const FtArgs& a) {
  const int wpg = a.log_g > 6 ? 1 << (a.log_g - 6) : 1;
  return 256 + up256((size_t)a.B * sizeof(float2)) + up256((size_t)a.B * sizeof(double)) + up256((size_t)a.B * a.wps * sizeof(double2)) +
         up256((size_t)a.B * a.wps * sizeof(int)) + up256((size_t)a.B * a.C * a.nseg * wpg * sizeof(double2));
}
void ft_carve(FtArgs* a, void* ws) {
  unsigned char* p = (unsigned char*)ws;
  a->total = (double*)p; a->late = (int*)(p + 128); p += 256;
  a->coef = (float2*)p; p += up256((size_t)a->B * sizeof(float2));
  a->term = (double*)p; p += up256((size_t)a->B * sizeof(double));
  a->part = (double2*)p; p += up256((size_t)a->B * a->wps * sizeof(double2));
  a->done = (int*)p; p += up256((size_t)a->B * a->wps * sizeof(int));
  a->chan = (double2*)p;
}
static double ft_bytes(const FtArgs& a, int mode, int dt, bool grad) {
  const double n = (double)a.B * a.C * (double)a.T;
  return n * (dt_size(dt) * (1.0 + (a.ref ? 1 : 0) * (!grad || mode == FT_POLICY ? 1 : 0) + (grad ? 1 : 0)) + (a.x ? 4.0 : 0.0) + 4.0 * a.second_rows / a.B);
}
int launch_ft_sums(const FtArgs& a, int mode, int dt, hipStream_t s) {
  PROF_SCOPE(mode == FT_PREF ? "pref_loss" : "policy_loss", 0, ft_bytes(a, mode, dt, false), s);
  if (mode == FT_PREF) return a.logit ? launch_sums_t<FT_PREF, true, true>(a, dt, s) : launch_sums_t<FT_PREF, false, true>(a, dt, s);
  if (a.ref) return a.logit ? launch_sums_t<FT_POLICY, true, true>(a, dt, s) : launch_sums_t<FT_POLICY, false, true>(a, dt, s);
  return a.logit ? launch_sums_t<FT_POLICY, true, false>(a, dt, s) : launch_sums_t<FT_POLICY, false, false>(a, dt, s);
}
int launch_ft_scale(const float* dloss, void* g, int dt, int64_t n, float* d_logit, int C, hipStream_t s) {
  const dim3 grid((unsigned)std::min<int64_t>(cdiv64(n, 4 * FT_THREADS), 2048));
  if (dt == DT_F32) hipLaunchKernelGGL((scale_kernel<float>), grid, dim3(FT_THREADS), 0, s, dloss, (float*)g, n, d_logit, C);
  else hipLaunchKernelGGL((scale_kernel<bf16_t>), grid, dim3(FT_THREADS), 0, s, dloss, (bf16_t*)g, n, d_logit, C);
  HIP_TRY(hipGetLastError());
  return DDMI_OK;
}
// the preference gradient does not need the reference's output: its residual is the trained network's alone
int launch_ft_grad(const FtArgs& a, int mode, int dt, hipStream_t s) {
  PROF_SCOPE(mode == FT_PREF ? "pref_loss_bwd" : "policy_loss_bwd", 0, ft_bytes(a, mode, dt, true), s);
  if (mode == FT_PREF) return a.logit ? launch_grad_t<FT_PREF, true, false>(a, dt, s) : launch_grad_t<FT_PREF, false, false>(a, dt, s);
  if (a.ref) return a.logit ? launch_grad_t<FT_POLICY, true, true>(a, dt, s) : launch_grad_t<FT_POLICY, false, true>(a, dt, s);
  return a.logit ? launch_grad_t<FT_POLICY, true, false>(a, dt, s) : launch_grad_t<FT_POLICY, false, false>(a, dt, s);
}
