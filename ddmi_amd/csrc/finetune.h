// The fine-tuning losses' kernels (k_finetune.hip) as the C entry points (finetune_capi.hip) see them.
#pragma once
#include "common.h"

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));            // rows of an odd plane, tensors of a slab start at any element
typedef unsigned short u16x4u __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned u32u __attribute__((aligned(1)));
// NT: past the caches, for streams of which nothing is found there again.
// (overloads, not a template: a deduced type would lose its alignment)
#define FT_GET_PUT(V)                                                                                   \
  template <bool NT> __device__ __forceinline__ V get(const V* p) {                                     \
    if constexpr (NT) return __builtin_nontemporal_load(p);                                             \
    else return *p;                                                                                     \
  }                                                                                                     \
  template <bool NT> __device__ __forceinline__ void put(V* p, V v) {                                   \
    if constexpr (NT) __builtin_nontemporal_store(v, p);                                                \
    else *p = v;                                                                                        \
  }
FT_GET_PUT(f32x4u)
FT_GET_PUT(u16x4u)
FT_GET_PUT(u32u)

enum { FT_PREF = 0, FT_POLICY = 1 };
#define FT_THREADS 256
#define FT_VECS 16       // vectors of four residuals that a thread of the one-pass kernel keeps in registers
#define FT_CACHE_BYTES 268435456.0   // the last-level cache: an optimizer step that touches more goes past it
#define FT_MOST_GROUPS ((1ll << 24) - 1)   // workgroups of 256 threads in one launch: below 2^32 threads
#define FT_ROWS 512      // most rows (sample, channel) of one workgroup: their mixing coefficients sit in LDS

struct FtArgs {
  // inputs; `second` is the noise (preference; second_rows = pairs when both of a pair share it) or the chain's next state (policy)
  const void* out;
  const void* ref;
  const float* x;
  const float* second;
  int second_rows;
  const float* s1;           // sqrt(1 - abar_t) a sample
  const float* logit;
  const float* ref_logit;
  const float* weight;       // a pair / transition; not > 0: left out, its values are not read
  const float* transition;   // [B][3]: mean = A x_t + E eps, standard deviation
  const float* logp_old;
  const float* advantage;
  double beta, smoothing, clip, kl_coef;
  // outputs
  float* loss;
  float* row_out[3];         // margin, mse | logp, ratio, kl
  const float* dloss;        // upstream gradient, a device scalar (null: 1)
  void* d_out;
  float* d_logit;
  // plan
  int B, C, pairs;
  int64_t T, seg;
  int wps, rows_per_wg, nseg, log_g, fused, polls;
  int again;                 // gradients of a call that has run, from its workspace, unless the upstream gradient is 1
  // workspace
  double* total;             // sum of the weights
  int* done;                 // one pass: whether a span's gradient is written
  int* late;                 // one pass: whether a workgroup has waited in vain
  float2* coef;              // a sample: factors of the residual and of the step away from the reference
  double* term;
  double2* part;             // a workgroup of sums_kernel
  double2* chan;             // a (sample, channel, segment, wave): sums the mixing logit's gradient needs
};
// rows_of: samples whose sums meet (2: a pair); keep: vectors a thread may keep for one pass over the inputs, 0: two passes; units: compute units
// of the card, FT_ANY_CARD: one pass wherever a card of some size would take it (to size a workspace)
#define FT_ANY_CARD -1
int ft_plan(FtArgs* a, int B, int C, int64_t HW, bool mixed, int rows_of, int keep, int units);
int ft_units();              // of the current device, 0 where there is none
size_t ft_workspace_bytes(const FtArgs& a);
void ft_carve(FtArgs* a, void* ws);
void ft_set_polls(int n);
int launch_ft_sums(const FtArgs& a, int mode, int dt, hipStream_t s);
int launch_ft_scale(const float* dloss, void* g, int dt, int64_t n, float* d_logit, int C, hipStream_t s);
int launch_ft_grad(const FtArgs& a, int mode, int dt, hipStream_t s);

#define ADAMW_BLOCK 256      // values of a tensor that share one scale of the 8-bit moments
int launch_adamw_multi(const ddmi_adamw_tensor* t, int n, double beta1, double beta2, double eps, double grad_scale, unsigned seed, int pdt, int gdt,
                       int state_bits, hipStream_t s);
