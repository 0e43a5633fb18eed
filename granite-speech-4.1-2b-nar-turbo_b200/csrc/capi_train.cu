// extern "C" entry points of the fine-tuning operators (declared in include/gsn_conv.h): argument checks and launches.
#include <math.h>

#include "gsn_conv.h"
#include "gsn_kernels.cuh"

using namespace gsn;

namespace {

int type_size(int dtype) { return dtype == GSN_FP32 ? 4 : 2; }

// returns -1 for a valid problem without rows, 0 to launch, or a GSN_ERR_* code
int check_rows(const char* name, int64_t M, int D, int dtype, const int32_t* lengths, int T) {
  if (M < 0 || D <= 0) return fail(GSN_ERR_INVALID_ARG, "%s: bad sizes M=%lld D=%d", name, (long long)M, D);
  if (M > 0x7fffffffLL) return fail(GSN_ERR_UNSUPPORTED, "%s: M=%lld rows, at most 2^31 - 1", name, (long long)M);
  if (D > kMaxRowElements) return fail(GSN_ERR_UNSUPPORTED, "%s: D=%d, at most %d", name, D, kMaxRowElements);
  if (dtype != GSN_BF16 && dtype != GSN_FP16 && dtype != GSN_FP32)
    return fail(GSN_ERR_UNSUPPORTED, "%s: dtype %d is none of bf16, fp16, fp32", name, dtype);
  if (lengths && M > 0 && (T <= 0 || M % T != 0))
    return fail(GSN_ERR_UNSUPPORTED, "%s: with lengths, T=%d must divide M=%lld", name, T, (long long)M);
  return M == 0 ? -1 : 0;
}

// a row operand: its pointer, and its stride at least the row
int check_operand(const char* name, const char* what, const void* p, int64_t ld, int D, int dtype) {
  if (!p) return fail(GSN_ERR_INVALID_ARG, "%s: null %s", name, what);
  if (ld < D) return fail(GSN_ERR_UNSUPPORTED, "%s: row stride %lld of %s below D=%d", name, (long long)ld, what, D);
  if (!aligned(p, type_size(dtype))) return fail(GSN_ERR_UNSUPPORTED, "%s: %s is not aligned to its type", name, what);
  return 0;
}

int check_params(const char* name, int D, int dtype, int param_dtype, const void* weight, const void* other) {
  if (D > kMaxRowWidth) return fail(GSN_ERR_UNSUPPORTED, "%s: D=%d, at most %d", name, D, kMaxRowWidth);
  if (param_dtype != GSN_FP32 && param_dtype != dtype)
    return fail(GSN_ERR_UNSUPPORTED, "%s: parameters of type %d, need fp32 or the rows' type %d", name, param_dtype,
                dtype);
  if (!weight || !other) return fail(GSN_ERR_INVALID_ARG, "%s: null parameter", name);
  if (!aligned(weight, type_size(param_dtype)) || !aligned(other, type_size(param_dtype)))
    return fail(GSN_ERR_UNSUPPORTED, "%s: parameters are not aligned to their type", name);
  return 0;
}

// of 65536 numbers, those below it drop; what remains is multiplied by the factor
uint32_t dropout_threshold(double p) { return (uint32_t)nearbyint(p * 65536.0); }

float dropout_factor(double p, double scale) {
  const uint32_t threshold = dropout_threshold(p);
  return threshold > 65535u ? 0.f : (float)(scale * 65536.0 / (65536.0 - threshold));
}

int check_dropout(const char* name, const int64_t* rng, double p, double scale) {
  if (!rng || !aligned(rng, 8)) return fail(GSN_ERR_INVALID_ARG, "%s: rng must be a device int64[2]", name);
  if (!(p >= 0.0 && p <= 1.0)) return fail(GSN_ERR_INVALID_ARG, "%s: p=%g is not a probability", name, p);
  if (!isfinite(scale) || !isfinite(dropout_factor(p, scale)))
    return fail(GSN_ERR_INVALID_ARG, "%s: scale=%g with p=%g is not finite in fp32", name, scale, p);
  return 0;
}

void set_dropout(RowArgs& a, const int64_t* rng, uint32_t site, double p, double scale) {
  a.rng = rng;
  a.site = site;
  a.threshold = dropout_threshold(p);
  a.drop_all = a.threshold > 65535u;
  a.factor = dropout_factor(p, scale);
}

RowArgs row_args(int64_t M, int D, float eps, const int32_t* lengths, int T, int param_dtype) {
  RowArgs a;
  a.M = M;
  a.D = D;
  a.groups = (D + 7) / 8;
  a.eps = eps;
  a.lengths = lengths;
  a.T = T;
  a.param_fp32 = param_dtype == GSN_FP32;
  return a;
}

int set_partials(const char* name, RowArgs& a, void* workspace, size_t bytes) {
  const size_t need = gsn_layer_norm_bwd_workspace_bytes(a.M, a.D);
  if (bytes < need) return fail(GSN_ERR_WORKSPACE, "%s: workspace %zu < %zu bytes", name, bytes, need);
  if (need && (!workspace || !aligned(workspace, 16)))
    return fail(GSN_ERR_INVALID_ARG, "%s: workspace must be 16-byte aligned", name);
  a.partials = static_cast<float*>(workspace);
  a.partial_rows = a.M > 0 ? row_partial_rows(a.M, a.D) : 0;
  return 0;
}

int check_ctc(const char* name, int B, int T, int V, int S, int64_t ld_b, int64_t ld_t, int blank, int dtype) {
  if (B < 0 || T < 0 || V <= 0 || S < 0) return fail(GSN_ERR_INVALID_ARG, "%s: B=%d T=%d V=%d S=%d", name, B, T, V, S);
  if (dtype != GSN_BF16 && dtype != GSN_FP16 && dtype != GSN_FP32)
    return fail(GSN_ERR_UNSUPPORTED, "%s: dtype %d is none of bf16, fp16, fp32", name, dtype);
  if (blank < 0 || blank >= V) return fail(GSN_ERR_INVALID_ARG, "%s: blank=%d outside the %d classes", name, blank, V);
  if (V > kMaxCtcClasses) return fail(GSN_ERR_UNSUPPORTED, "%s: V=%d classes, at most %d", name, V, kMaxCtcClasses);
  if (S > kMaxCtcLabels) return fail(GSN_ERR_UNSUPPORTED, "%s: S=%d labels, at most %d", name, S, kMaxCtcLabels);
  if (T > kMaxCtcFrames) return fail(GSN_ERR_UNSUPPORTED, "%s: T=%d frames, at most %d", name, T, kMaxCtcFrames);
  if (B * (int64_t)T > 0 && (ld_t < V || ld_b < 0))
    return fail(GSN_ERR_UNSUPPORTED, "%s: strides %lld, %lld of logits", name, (long long)ld_b, (long long)ld_t);
  return B == 0 ? -1 : 0;
}

CtcArgs ctc_args(const void* logits, int64_t ld_b, int64_t ld_t, const int32_t* targets, const int32_t* input_lengths,
                 const int32_t* target_lengths, int B, int T, int V, int S, int blank, int zero_infinity) {
  CtcArgs a;
  a.logits = logits;
  a.ld_b = ld_b;
  a.ld_t = ld_t;
  a.targets = targets;
  a.input_lengths = input_lengths;
  a.target_lengths = target_lengths;
  a.B = B;
  a.T = T;
  a.V = V;
  a.S = S;
  a.blank = blank;
  a.zero_infinity = zero_infinity;
  a.pitch = ctc_pitch(S);
  a.state_pitch = ctc_state_pitch(S);
  return a;
}

// what the forward pass leaves for the backward pass, in one buffer
int set_state(const char* name, CtcArgs& a, void* state, size_t bytes) {
  const size_t need = gsn_ctc_loss_state_bytes(a.B, a.T, a.S);
  if (bytes < need) return fail(GSN_ERR_WORKSPACE, "%s: state %zu < %zu bytes", name, bytes, need);
  if (!state || !aligned(state, 16)) return fail(GSN_ERR_INVALID_ARG, "%s: state must be 16-byte aligned", name);
  char* p = static_cast<char*>(state);
  a.raw_loss = (float*)p;
  p += align256(a.B * sizeof(float));
  a.again = (int*)p;
  p += align256(a.B * sizeof(int));
  a.stats = (float2*)p;
  p += align256((size_t)a.B * a.T * sizeof(float2));
  a.order = (int2*)p;
  p += align256((size_t)a.B * a.pitch * sizeof(int2));
  a.post = (float*)p;
  return 0;
}

// gsn_ctc_loss_fwd, or with a copy withheld for the self-test
int ctc_loss_fwd(const char* name, const void* logits, int64_t ld_b, int64_t ld_t, const int32_t* targets,
                 const int32_t* input_lengths, const int32_t* target_lengths, int B, int T, int V, int S, int blank,
                 int zero_infinity, int gradient, int dtype, float* loss, void* state, size_t state_bytes, void* workspace,
                 size_t workspace_bytes, int withhold, gsn_stream_t stream) {
  if (int rc = check_ctc(name, B, T, V, S, ld_b, ld_t, blank, dtype)) return rc < 0 ? ok() : rc;
  if (!input_lengths || !target_lengths || !loss || (S > 0 && !targets) || (T > 0 && !logits))
    return fail(GSN_ERR_INVALID_ARG, "%s: null pointer", name);
  if (!aligned(logits, type_size(dtype))) return fail(GSN_ERR_UNSUPPORTED, "%s: logits are not aligned to their type", name);
  CtcArgs a = ctc_args(logits, ld_b, ld_t, targets, input_lengths, target_lengths, B, T, V, S, blank, zero_infinity);
  if (int rc = set_state(name, a, state, state_bytes)) return rc;
  const size_t need = gsn_ctc_loss_workspace_bytes(B, T, S, gradient);
  if (workspace_bytes < need) return fail(GSN_ERR_WORKSPACE, "%s: workspace %zu < %zu bytes", name, workspace_bytes, need);
  if (!workspace || !aligned(workspace, 16)) return fail(GSN_ERR_INVALID_ARG, "%s: workspace must be 16-byte aligned", name);
  a.loss = loss;
  a.withhold = withhold;
  char* ws = static_cast<char*>(workspace);
  a.bad = (int*)ws;
  ws += align256((size_t)B * sizeof(int));
  a.norms = (float*)ws;
  ws += align256((size_t)B * T * sizeof(float));
  a.exchange = (float2*)ws;
  if (gradient) {
    a.states = (uint32_t*)(ws + align256((size_t)B * 8 * a.pitch * sizeof(float2)));
    a.upper = a.states + (size_t)B * T * a.state_pitch;
  }
  return finish(launch_ctc_loss(a, dtype, (cudaStream_t)stream), name);
}

}  // namespace

extern "C" {

int gsn_layer_norm_fwd(const void* x, int64_t ld_x, const void* weight, const void* bias, void* y, int64_t M, int D,
                       float eps, int dtype, int param_dtype, const int32_t* lengths, int T, gsn_stream_t stream) {
  const char* name = "gsn_layer_norm_fwd";
  if (int rc = check_rows(name, M, D, dtype, lengths, T)) return rc < 0 ? ok() : rc;
  if (int rc = check_params(name, D, dtype, param_dtype, weight, bias)) return rc;
  if (int rc = check_operand(name, "x", x, ld_x, D, dtype)) return rc;
  if (int rc = check_operand(name, "y", y, D, D, dtype)) return rc;
  RowArgs a = row_args(M, D, eps, lengths, T, param_dtype);
  a.x = x;
  a.ld_x = ld_x;
  a.weight = weight;
  a.bias = bias;
  a.y = y;
  return finish(launch_row_op(a, kRowNorm, dtype, (cudaStream_t)stream), name);
}

size_t gsn_layer_norm_bwd_workspace_bytes(int64_t M, int D) {
  if (M <= 0 || D <= 0 || M > 0x7fffffffLL || D > kMaxRowWidth) return 0;
  return (size_t)row_partial_rows(M, D) * 2 * D * sizeof(float);
}

int gsn_layer_norm_bwd(const void* dy, int64_t ld_dy, const void* x, int64_t ld_x, const void* weight, void* dx,
                       void* dweight, void* dbias, int64_t M, int D, float eps, int dtype, int param_dtype,
                       const int32_t* lengths, int T, void* workspace, size_t workspace_bytes, gsn_stream_t stream) {
  const char* name = "gsn_layer_norm_bwd";
  const int empty = check_rows(name, M, D, dtype, lengths, T);
  if (empty > 0) return empty;
  if (int rc = check_params(name, D, dtype, param_dtype, weight, dweight)) return rc;
  if (!dbias || !aligned(dbias, type_size(param_dtype))) return fail(GSN_ERR_INVALID_ARG, "%s: dbias", name);
  RowArgs a = row_args(M, D, eps, lengths, T, param_dtype);
  if (!empty) {
    if (int rc = check_operand(name, "dy", dy, ld_dy, D, dtype)) return rc;
    if (int rc = check_operand(name, "x", x, ld_x, D, dtype)) return rc;
    if (int rc = check_operand(name, "dx", dx, D, D, dtype)) return rc;
    if (int rc = set_partials(name, a, workspace, workspace_bytes)) return rc;
  }
  a.x = x;
  a.ld_x = ld_x;
  a.dy = dy;
  a.ld_dy = ld_dy;
  a.weight = weight;
  a.dx = dx;
  a.dweight = dweight;
  a.dbias = dbias;
  return finish(launch_row_op(a, kRowNormGrad, dtype, (cudaStream_t)stream), name);
}

int gsn_dropout_add(const void* x, int64_t ld_x, const void* residual, int64_t ld_res, void* out, int64_t M, int D,
                    int dtype, const int64_t* rng, uint32_t site, double p, double scale, const int32_t* lengths, int T,
                    gsn_stream_t stream) {
  const char* name = "gsn_dropout_add";
  if (int rc = check_rows(name, M, D, dtype, lengths, T)) return rc < 0 ? ok() : rc;
  if (int rc = check_dropout(name, rng, p, scale)) return rc;
  if (int rc = check_operand(name, "x", x, ld_x, D, dtype)) return rc;
  if (residual)
    if (int rc = check_operand(name, "residual", residual, ld_res, D, dtype)) return rc;
  if (int rc = check_operand(name, "out", out, D, D, dtype)) return rc;
  RowArgs a = row_args(M, D, 0.f, lengths, T, dtype);
  a.x = x;
  a.ld_x = ld_x;
  a.residual = residual;
  a.ld_res = residual ? ld_res : 0;
  a.y = out;
  set_dropout(a, rng, site, p, scale);
  return finish(launch_row_op(a, kRowDropout, dtype, (cudaStream_t)stream), name);
}

int gsn_dropout_add_layer_norm_fwd(const void* x, int64_t ld_x, const void* residual, int64_t ld_res,
                                   const void* weight, const void* bias, void* y, void* h, int64_t M, int D, float eps,
                                   int dtype, int param_dtype, const int64_t* rng, uint32_t site, double p,
                                   double scale, const int32_t* lengths, int T, gsn_stream_t stream) {
  const char* name = "gsn_dropout_add_layer_norm_fwd";
  if (int rc = check_rows(name, M, D, dtype, lengths, T)) return rc < 0 ? ok() : rc;
  if (int rc = check_params(name, D, dtype, param_dtype, weight, bias)) return rc;
  if (int rc = check_dropout(name, rng, p, scale)) return rc;
  if (int rc = check_operand(name, "x", x, ld_x, D, dtype)) return rc;
  if (int rc = check_operand(name, "residual", residual, ld_res, D, dtype)) return rc;
  if (int rc = check_operand(name, "y", y, D, D, dtype)) return rc;
  if (int rc = check_operand(name, "h", h, D, D, dtype)) return rc;
  RowArgs a = row_args(M, D, eps, lengths, T, param_dtype);
  a.x = x;
  a.ld_x = ld_x;
  a.residual = residual;
  a.ld_res = ld_res;
  a.weight = weight;
  a.bias = bias;
  a.y = y;
  a.h_out = h;
  set_dropout(a, rng, site, p, scale);
  return finish(launch_row_op(a, kRowDropNorm, dtype, (cudaStream_t)stream), name);
}

int gsn_dropout_add_layer_norm_bwd(const void* dy, int64_t ld_dy, const void* dh, int64_t ld_dh, const void* h,
                                   int64_t ld_h, const void* weight, void* dx, void* dresidual, void* dweight,
                                   void* dbias, int64_t M, int D, float eps, int dtype, int param_dtype,
                                   const int64_t* rng, uint32_t site, double p, double scale, const int32_t* lengths,
                                   int T, void* workspace, size_t workspace_bytes, gsn_stream_t stream) {
  const char* name = "gsn_dropout_add_layer_norm_bwd";
  const int empty = check_rows(name, M, D, dtype, lengths, T);
  if (empty > 0) return empty;
  if (int rc = check_params(name, D, dtype, param_dtype, weight, dweight)) return rc;
  if (!dbias || !aligned(dbias, type_size(param_dtype))) return fail(GSN_ERR_INVALID_ARG, "%s: dbias", name);
  if (int rc = check_dropout(name, rng, p, scale)) return rc;
  RowArgs a = row_args(M, D, eps, lengths, T, param_dtype);
  if (!empty) {
    if (int rc = check_operand(name, "dy", dy, ld_dy, D, dtype)) return rc;
    if (dh)
      if (int rc = check_operand(name, "dh", dh, ld_dh, D, dtype)) return rc;
    if (int rc = check_operand(name, "h", h, ld_h, D, dtype)) return rc;
    if (int rc = check_operand(name, "dx", dx, D, D, dtype)) return rc;
    if (int rc = check_operand(name, "dresidual", dresidual, D, D, dtype)) return rc;
    if (int rc = set_partials(name, a, workspace, workspace_bytes)) return rc;
  }
  a.x = h;
  a.ld_x = ld_h;
  a.dy = dy;
  a.ld_dy = ld_dy;
  a.dh = dh;
  a.ld_dh = dh ? ld_dh : 0;
  a.weight = weight;
  a.dx = dx;
  a.dres = dresidual;
  a.dweight = dweight;
  a.dbias = dbias;
  set_dropout(a, rng, site, p, scale);
  return finish(launch_row_op(a, kRowDropNormGrad, dtype, (cudaStream_t)stream), name);
}

size_t gsn_ctc_loss_state_bytes(int B, int T, int S) {
  if (B <= 0 || T < 0 || S < 0 || S > kMaxCtcLabels) return 0;
  const size_t frames = (size_t)B * T, pitch = ctc_pitch(S);
  return align256(B * sizeof(float)) + align256(B * sizeof(int)) + align256(frames * sizeof(float2)) + align256(B * pitch * sizeof(int2)) +
         align256(frames * pitch * sizeof(float));
}

size_t gsn_ctc_loss_workspace_bytes(int B, int T, int S, int gradient) {
  if (B <= 0 || T < 0 || S < 0 || S > kMaxCtcLabels) return 0;
  size_t n = align256((size_t)B * sizeof(int)) + align256((size_t)B * T * sizeof(float)) +
             align256((size_t)B * 8 * ctc_pitch(S) * sizeof(float2));
  if (gradient) n += (size_t)B * T * (ctc_state_pitch(S) + ctc_pitch(S)) * sizeof(uint32_t);
  return n;
}

int gsn_ctc_loss_fwd(const void* logits, int64_t ld_b, int64_t ld_t, const int32_t* targets,
                     const int32_t* input_lengths, const int32_t* target_lengths, int B, int T, int V, int S, int blank,
                     int zero_infinity, int gradient, int dtype, float* loss, void* state, size_t state_bytes,
                     void* workspace, size_t workspace_bytes, gsn_stream_t stream) {
  return ctc_loss_fwd("gsn_ctc_loss_fwd", logits, ld_b, ld_t, targets, input_lengths, target_lengths, B, T, V, S, blank,
                      zero_infinity, gradient, dtype, loss, state, state_bytes, workspace, workspace_bytes, 0, stream);
}

int gsn_selftest_ctc_withheld(const void* logits, int64_t ld_b, int64_t ld_t, const int32_t* targets,
                              const int32_t* input_lengths, const int32_t* target_lengths, int B, int T, int V, int S,
                              int blank, int dtype, float* loss, void* state, size_t state_bytes, void* workspace,
                              size_t workspace_bytes, int side, int half, gsn_stream_t stream) {
  const char* name = "gsn_selftest_ctc_withheld";
  if (side < 0 || side > 1 || half < 0 || half > 1) return fail(GSN_ERR_INVALID_ARG, "%s: side=%d half=%d", name, side, half);
  if (S > kMaxCtcHeldLabels) return fail(GSN_ERR_UNSUPPORTED, "%s: S=%d labels, at most %d", name, S, kMaxCtcHeldLabels);
  return ctc_loss_fwd(name, logits, ld_b, ld_t, targets, input_lengths, target_lengths, B, T, V, S, blank, 0, 1, dtype,
                      loss, state, state_bytes, workspace, workspace_bytes, 1 + side + 2 * half, stream);
}

int gsn_ctc_loss_bwd(const float* dloss, const void* logits, int64_t ld_b, int64_t ld_t, const int32_t* targets,
                     const int32_t* input_lengths, const int32_t* target_lengths, int B, int T, int V, int S, int blank,
                     int zero_infinity, int dtype, const void* state, size_t state_bytes, void* dlogits,
                     gsn_stream_t stream) {
  const char* name = "gsn_ctc_loss_bwd";
  if (int rc = check_ctc(name, B, T, V, S, ld_b, ld_t, blank, dtype)) return rc < 0 ? ok() : rc;
  if (T == 0) return ok();
  if (!dloss || !logits || !input_lengths || !target_lengths || (S > 0 && !targets) || !dlogits)
    return fail(GSN_ERR_INVALID_ARG, "%s: null pointer", name);
  if (!aligned(logits, type_size(dtype)) || !aligned(dlogits, type_size(dtype)))
    return fail(GSN_ERR_UNSUPPORTED, "%s: logits and dlogits are not aligned to their type", name);
  CtcArgs a = ctc_args(logits, ld_b, ld_t, targets, input_lengths, target_lengths, B, T, V, S, blank, zero_infinity);
  if (int rc = set_state(name, a, const_cast<void*>(state), state_bytes)) return rc;
  a.dloss = dloss;
  a.dlogits = dlogits;
  return finish(launch_ctc_grad(a, dtype, (cudaStream_t)stream), name);
}

}  // extern "C"
