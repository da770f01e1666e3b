// C ABI of the fine-tuning operators (include/ddmi_hip.h, "Fine-tuning"): no handle, no state; the caller owns every buffer, the losses'
// workspace among them (so two captured graphs, or two streams, that use workspaces of their own share nothing).
#include <algorithm>
#include <cmath>
#include <initializer_list>
#include "finetune.h"

namespace {
bool dtype_ok(int dt) { return dt == DDMI_DTYPE_F32 || dt == DDMI_DTYPE_BF16; }
int internal_dt(int dt) { return dt == DDMI_DTYPE_F32 ? DT_F32 : DT_BF16; }

bool aligned(std::initializer_list<const void*> ps, int bytes) {      // null is
  for (const void* p : ps)
    if ((uintptr_t)p & (uintptr_t)(bytes - 1)) return false;
  return true;
}
int size_of(int dt) { return dt == DDMI_DTYPE_F32 ? 4 : 2; }

int common_args(FtArgs* a, const ddmi_loss_in* in, int B, int rows_of, int keep, void* ws, size_t ws_bytes) {
  DDMI_REQUIRE(in->model_out && in->second && B > 0 && in->C > 0 && in->HW > 0, "fine-tuning loss: null argument or empty batch");
  DDMI_REQUIRE(dtype_ok(in->out_dtype), "fine-tuning loss: model_out / ref_out are fp32 or bf16");
  DDMI_REQUIRE((in->mixing_logit == nullptr) == (in->ref_mixing_logit == nullptr) || (in->mixing_logit && !in->ref_out), "fine-tuning loss: both mixing logits or none");
  DDMI_REQUIRE(!in->mixing_logit || (in->x_t && in->sqrt_1mac), "fine-tuning loss: mixing needs x_t and sqrt_1mac");
  DDMI_REQUIRE(aligned({in->model_out, in->ref_out}, size_of(in->out_dtype)) &&
                   aligned({in->x_t, in->second, in->sqrt_1mac, in->mixing_logit, in->ref_mixing_logit, in->weight}, 4),
               "fine-tuning loss: inputs aligned to their values");
  DDMI_REQUIRE((double)in->C * (double)in->HW < 1.1e12, "fine-tuning loss: sample too large");
  DDMI_TRY(ft_plan(a, B, in->C, in->HW, in->mixing_logit != nullptr, rows_of, keep, ft_units()));
  DDMI_REQUIRE(ws && ((uintptr_t)ws & 15) == 0 && ws_bytes >= ft_workspace_bytes(*a), "fine-tuning loss: workspace too small or not 16-byte aligned");
  ft_carve(a, ws);
  a->out = in->model_out; a->ref = in->ref_out; a->x = in->x_t; a->second = in->second; a->s1 = in->mixing_logit ? in->sqrt_1mac : nullptr;
  a->logit = in->mixing_logit; a->ref_logit = in->ref_mixing_logit; a->weight = in->weight;
  return DDMI_OK;
}
// vectors a thread of the one-pass form keeps
int kept(int mode, const ddmi_loss_in* in) { return mode == FT_POLICY && in->ref_out ? FT_VECS / 2 : FT_VECS; }
int run(FtArgs* a, int mode, int out_dtype, hipStream_t s) {
  DDMI_TRY(launch_ft_sums(*a, mode, internal_dt(out_dtype), s));
  return a->d_out ? launch_ft_grad(*a, mode, internal_dt(out_dtype), s) : DDMI_OK;
}
}  // namespace

extern "C" {

int ddmi_train_loss_workspace_bytes(int B, int C, int64_t HW, int mixed, size_t* bytes) {
  DDMI_REQUIRE(bytes && B > 0 && C > 0 && HW > 0 && (double)C * (double)HW < 1.1e12, "train_loss_workspace_bytes: bad arguments");
  *bytes = 0;
  for (int rows_of = 1; rows_of <= 2; ++rows_of)
    for (int keep : {0, FT_VECS / 2, FT_VECS}) {      // whichever loss the call is, with or without its gradient, on whichever card
      FtArgs a{};
      DDMI_TRY(ft_plan(&a, B, C, HW, mixed != 0, rows_of, keep, FT_ANY_CARD));
      *bytes = std::max(*bytes, ft_workspace_bytes(a));
    }
  return DDMI_OK;
}

int ddmi_train_pref_loss(const ddmi_loss_in* in, int pairs, int noise_rows, double beta, double label_smoothing, const float* dloss, void* ws,
                         size_t ws_bytes, float* loss, float* margin, float* mse, void* d_model_out, float* d_logit, void* stream) {
  FtArgs a{};
  DDMI_REQUIRE(in && in->ref_out && pairs > 0 && pairs <= (1 << 24), "pref_loss: null argument or no pairs");
  DDMI_REQUIRE(loss && margin && mse, "pref_loss: null output");
  DDMI_REQUIRE(noise_rows == pairs || noise_rows == 2 * pairs, "pref_loss: the noise has a row for each pair or for each sample");
  DDMI_REQUIRE(label_smoothing >= 0.0 && label_smoothing <= 1.0 && std::isfinite(beta), "pref_loss: label_smoothing in [0, 1], beta finite");
  DDMI_REQUIRE(!d_logit || (in->mixing_logit && d_model_out), "pref_loss: d_logit goes with mixing_logit and d_model_out");
  DDMI_REQUIRE(aligned({loss, margin, mse, dloss, d_logit}, 4) && aligned({d_model_out}, size_of(in->out_dtype)), "pref_loss: outputs aligned to their values");
  DDMI_TRY(common_args(&a, in, 2 * pairs, 2, d_model_out ? kept(FT_PREF, in) : 0, ws, ws_bytes));
  if (!in->mixing_logit) a.x = nullptr;      // not read
  a.pairs = pairs; a.second_rows = noise_rows; a.beta = beta; a.smoothing = label_smoothing;
  a.loss = loss; a.row_out[0] = margin; a.row_out[1] = mse; a.dloss = dloss; a.d_out = d_model_out; a.d_logit = d_logit;
  return run(&a, FT_PREF, in->out_dtype, (hipStream_t)stream);
}
int ddmi_train_policy_loss(const ddmi_loss_in* in, int B, const float* transition, const float* logp_old, const float* advantage, double clip_range,
                           double kl_coef, const float* dloss, void* ws, size_t ws_bytes, float* loss, float* logp, float* ratio, float* kl,
                           void* d_model_out, float* d_logit, void* stream) {
  FtArgs a{};
  DDMI_REQUIRE(in && transition && in->x_t && logp, "policy_loss: null argument");
  DDMI_REQUIRE(!logp_old || (advantage && loss && ratio && kl), "policy_loss: null argument");
  DDMI_REQUIRE(clip_range >= 0.0 && std::isfinite(kl_coef), "policy_loss: clip_range >= 0, kl_coef finite");
  DDMI_REQUIRE(kl_coef == 0.0 || in->ref_out, "policy_loss: a KL term needs the reference's output");
  DDMI_REQUIRE(logp_old || !d_model_out, "policy_loss: a gradient of the log-density alone is not offered");
  DDMI_REQUIRE(!d_logit || (in->mixing_logit && d_model_out), "policy_loss: d_logit goes with mixing_logit and d_model_out");
  DDMI_REQUIRE(aligned({transition, logp_old, advantage, loss, logp, ratio, kl, dloss, d_logit}, 4) && aligned({d_model_out}, size_of(in->out_dtype)),
               "policy_loss: tensors aligned to their values");
  DDMI_TRY(common_args(&a, in, B, 1, d_model_out ? kept(FT_POLICY, in) : 0, ws, ws_bytes));
  a.pairs = B; a.second_rows = B; a.transition = transition;
  a.logp_old = logp_old; a.advantage = advantage; a.clip = clip_range; a.kl_coef = kl_coef;
  a.loss = logp_old ? loss : nullptr; a.row_out[0] = logp; a.row_out[1] = ratio; a.row_out[2] = kl;
  a.dloss = dloss; a.d_out = d_model_out; a.d_logit = d_logit;
  return run(&a, FT_POLICY, in->out_dtype, (hipStream_t)stream);
}
int ddmi_train_loss_scale(const float* dloss, void* d_model_out, int out_dtype, int64_t n, float* d_logit, int C, void* stream) {
  DDMI_REQUIRE(dloss && d_model_out && n > 0 && dtype_ok(out_dtype) && (!d_logit || C > 0), "loss_scale: bad arguments");
  DDMI_REQUIRE(aligned({dloss, d_logit}, 4) && aligned({d_model_out}, size_of(out_dtype)), "loss_scale: tensors aligned to their values");
  return launch_ft_scale(dloss, d_model_out, internal_dt(out_dtype), n, d_logit, C, (hipStream_t)stream);
}
int ddmi_train_loss_again(const ddmi_loss_in* in, int B, int noise_rows, const float* transition, const float* dloss, void* ws, size_t ws_bytes,
                          void* d_model_out, float* d_logit, void* stream) {
  const int mode = transition ? FT_POLICY : FT_PREF;
  FtArgs a{};
  DDMI_REQUIRE(in && dloss && d_model_out, "loss_again: null argument");
  DDMI_REQUIRE(transition ? in->x_t != nullptr : in->ref_out && B % 2 == 0 && (noise_rows == B / 2 || noise_rows == B), "loss_again: arguments of neither loss");
  DDMI_REQUIRE(!d_logit || in->mixing_logit, "loss_again: d_logit goes with mixing_logit");
  DDMI_REQUIRE(aligned({transition, dloss, d_logit}, 4) && aligned({d_model_out}, size_of(in->out_dtype)), "loss_again: tensors aligned to their values");
  DDMI_TRY(common_args(&a, in, B, transition ? 1 : 2, kept(mode, in), ws, ws_bytes));
  if (!transition && !in->mixing_logit) a.x = nullptr;      // not read
  a.pairs = transition ? B : B / 2; a.second_rows = transition ? B : noise_rows; a.transition = transition;
  a.dloss = dloss; a.d_out = d_model_out; a.d_logit = d_logit;
  a.fused = 0; a.again = 1;
  return launch_ft_grad(a, mode, internal_dt(in->out_dtype), (hipStream_t)stream);
}
int ddmi_stream_capture_id(void* stream, uint64_t* id) {
  DDMI_REQUIRE(id, "stream_capture_id: null argument");
  *id = 0;
  if (!stream) return DDMI_OK;      // the default stream is never captured
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  unsigned long long n = 0;
  HIP_TRY(hipStreamGetCaptureInfo((hipStream_t)stream, &status, &n));
  if (status == hipStreamCaptureStatusActive) *id = n;
  return DDMI_OK;
}
int ddmi_debug_loss_plan(int B, int C, int64_t HW, int mixed, int policy, int has_ref, int units, int* one_pass, int* spans) {
  DDMI_REQUIRE(one_pass && spans && B > 0 && C > 0 && HW > 0 && (double)C * (double)HW < 1.1e12 && units >= 0, "debug_loss_plan: bad arguments");
  FtArgs a{};
  DDMI_TRY(ft_plan(&a, B, C, HW, mixed != 0, policy ? 1 : 2, policy && has_ref ? FT_VECS / 2 : FT_VECS, units));
  *one_pass = a.fused;
  *spans = a.wps;
  return DDMI_OK;
}
int ddmi_debug_loss_polls(int n) {
  DDMI_REQUIRE(n >= 0, "debug_loss_polls: not negative");
  ft_set_polls(n);
  return DDMI_OK;
}

int ddmi_train_adamw_multi(const ddmi_adamw_tensor* tensors, int n, double beta1, double beta2, double eps, double grad_scale, uint32_t seed,
                           int param_dtype, int grad_dtype, int state_bits, void* stream) {
  DDMI_REQUIRE(n == 0 || (tensors && n > 0), "adamw_multi: null argument");
  DDMI_REQUIRE(dtype_ok(param_dtype) && dtype_ok(grad_dtype), "adamw_multi: parameters and gradients are fp32 or bf16");
  DDMI_REQUIRE(state_bits == 32 || state_bits == 8, "adamw_multi: moments have 32 or 8 bits");
  DDMI_REQUIRE(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0 && eps >= 0.0, "adamw_multi: betas in [0, 1), eps >= 0");
  for (int i = 0; i < n; ++i) {
    const ddmi_adamw_tensor& t = tensors[i];
    DDMI_REQUIRE(t.numel >= 0 && t.step >= 1, "adamw_multi: step counts from 1");
    if (t.numel == 0) continue;
    DDMI_REQUIRE(t.param && t.grad && t.exp_avg && t.exp_avg_sq, "adamw_multi: null tensor");
    DDMI_REQUIRE(state_bits == 32 || (t.exp_avg_scale && t.exp_avg_sq_scale), "adamw_multi: 8-bit moments need their scales");
    DDMI_REQUIRE(aligned({t.param}, size_of(param_dtype)) && aligned({t.grad}, size_of(grad_dtype)) &&
                     (state_bits == 32 ? aligned({t.exp_avg, t.exp_avg_sq}, 4) : aligned({t.exp_avg_scale, t.exp_avg_sq_scale}, 4)),
                 "adamw_multi: tensors aligned to their values");
  }
  return launch_adamw_multi(tensors, n, beta1, beta2, eps, grad_scale, seed, internal_dt(param_dtype), internal_dt(grad_dtype), state_bits,
                            (hipStream_t)stream);
}

}  // extern "C"
