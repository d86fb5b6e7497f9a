// C entry points of the conditioning calls: argument checks, then dispatch.
// The checks need no device, so a caller (and the CPU tests) can ask for a
// refusal's reason through the *_workspace_size calls.
#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdio>
#include <cstdlib>

#include "conditioning.cuh"

namespace {

using h3::Rows;

struct Refusal {
  h3c_status status = H3C_OK;
  std::string why;
  explicit operator bool() const { return status != H3C_OK; }
};

Refusal no(h3c_status st, const std::string& why) { return {st, why}; }

// Keeps the calling thread's current device.
struct DeviceGuard {
  int before = -1;
  cudaError_t err;
  explicit DeviceGuard(int device) {
    err = cudaGetDevice(&before);
    if (err == cudaSuccess && before != device) err = cudaSetDevice(device);
    else if (err == cudaSuccess) before = -1;
  }
  ~DeviceGuard() {
    if (before >= 0) cudaSetDevice(before);
  }
};

// a b c > limit, for 32-bit numbers that are not negative.
bool product_over(int64_t a, int64_t b, int64_t c, int64_t limit) { return c > 0 && (a * b > limit || a * b * c > limit); }

// Normalises one [batch, tokens, heads, 128] operand.  Outputs may not have
// two elements in one place.
Refusal rows(const h3c_bview& v, int64_t batch, int64_t tokens, int64_t heads, bool output, const char* name,
             Rows* r) {
  *r = {};
  if (batch == 0 || tokens == 0) return {};
  const std::string n = name;
  if (!v.ptr) return no(H3C_ERR_INVALID_ARGUMENT, n + " is null");
  struct Axis {
    int64_t size, stride;
  } ax[3] = {{batch, v.batch_stride}, {tokens, v.token_stride}, {heads, v.head_stride}};
  if ((uintptr_t)v.ptr & 15) return no(H3C_ERR_UNSUPPORTED, n + " needs 16-byte aligned rows");
  for (int i = 0; i < 3; ++i) {
    if (ax[i].size == 1) {
      ax[i].stride = 0;
      continue;
    }
    if (ax[i].stride < 0) return no(H3C_ERR_INVALID_ARGUMENT, n + " has a negative stride");
    if (ax[i].stride & 7) return no(H3C_ERR_UNSUPPORTED, n + " needs 16-byte aligned rows");
    if (ax[i].stride >= (int64_t)1 << 39) return no(H3C_ERR_UNSUPPORTED, n + " has a stride of 2^40 bytes or more");
    if (i == 1 && !output && ax[i].stride == 0)
      return no(H3C_ERR_UNSUPPORTED, n + " is broadcast over its tokens");
  }
  r->p = (uint16_t*)v.ptr;
  r->b = ax[0].stride;
  r->t = ax[1].stride;
  r->h = ax[2].stride;
  if (output) {
    std::sort(ax, ax + 3, [](const Axis& a, const Axis& b) { return a.stride < b.stride; });
    int64_t extent = 128;
    for (const Axis& a : ax) {
      if (a.size == 1) continue;
      if (a.stride < extent) return no(H3C_ERR_INVALID_ARGUMENT, n + " overlaps itself");
      if (a.stride > ((int64_t)1 << 46) / (a.size - 1)) return no(H3C_ERR_UNSUPPORTED, n + " spans 2^47 bytes or more");
      extent += (a.size - 1) * a.stride;
    }
  }
  return {};
}

#define H3_REFUSE(expr)        \
  do {                         \
    Refusal r_ = (expr);       \
    if (r_) return r_;         \
  } while (0)

Refusal check_cross(const h3c_cross_args* a, int op, h3::CrossLaunch* L) {
  if (!a) return no(H3C_ERR_INVALID_ARGUMENT, "null args");
  if (op < H3C_OP_CROSS_FWD || op > H3C_OP_PREFIX_FWD) return no(H3C_ERR_INVALID_ARGUMENT, "unknown operator");
  const bool bwd = op == H3C_OP_CROSS_BWD, prefix = op == H3C_OP_PREFIX_FWD;
  if (a->head_dim != 128) return no(H3C_ERR_UNSUPPORTED, "head_dim must be 128");
  if (a->batch < 0 || a->q_len < 0 || a->kv_len < 0 || a->heads <= 0 || a->kv_heads <= 0 || a->reserved != 0)
    return no(H3C_ERR_INVALID_ARGUMENT, "bad batch, lengths, heads or reserved");
  if (a->heads % a->kv_heads) return no(H3C_ERR_INVALID_ARGUMENT, "heads must be a multiple of kv_heads");
  if (!(a->scale > 0.f) || !std::isfinite(a->scale))
    return no(H3C_ERR_INVALID_ARGUMENT, "scale must be positive and finite");
  if (prefix && a->prefix_len < 0) return no(H3C_ERR_INVALID_ARGUMENT, "prefix_len must not be negative");
  const int64_t B = a->batch, P = prefix ? a->prefix_len : 0;
  // row and tile numbers are 32-bit in the kernels
  if (product_over(B, a->heads, std::max(a->q_len, 1), INT_MAX) ||
      product_over(B, a->heads, ((int64_t)a->kv_len + 127) / 128, INT_MAX) ||
      P + a->kv_len > INT_MAX - 256 || a->q_len > INT_MAX - 256)
    return no(H3C_ERR_UNSUPPORTED, "more than 2^31 rows");
  h3::CrossLaunch l{};
  l.n = {a->batch, a->q_len, a->kv_len, (int32_t)P, a->heads, a->kv_heads, a->heads / a->kv_heads};
  H3_REFUSE(rows(a->q, B, a->q_len, a->heads, false, "q", &l.q));
  H3_REFUSE(rows(a->out, B, a->q_len, a->heads, !bwd, "out", &l.out));
  H3_REFUSE(rows(a->k, B, a->kv_len, a->kv_heads, false, "k", &l.k));
  H3_REFUSE(rows(a->v, B, a->kv_len, a->kv_heads, false, "v", &l.v));
  if (prefix && B > 0) {
    H3_REFUSE(rows({a->prefix_k.ptr, 0, a->prefix_k.token_stride, a->prefix_k.head_stride}, 1, P, a->kv_heads, false,
                   "prefix_k", &l.pk));
    H3_REFUSE(rows({a->prefix_v.ptr, 0, a->prefix_v.token_stride, a->prefix_v.head_stride}, 1, P, a->kv_heads, false,
                   "prefix_v", &l.pv));
  }
  if (((uintptr_t)a->kv_lens & 3) || ((uintptr_t)a->lse & 3))
    return no(H3C_ERR_UNSUPPORTED, "kv_lens and lse need 4-byte alignment");
  if (bwd) {
    if (!a->lse && B > 0 && a->q_len > 0) return no(H3C_ERR_INVALID_ARGUMENT, "the backward call needs lse");
    H3_REFUSE(rows(a->out_grad, B, a->q_len, a->heads, false, "out_grad", &l.dout));
    H3_REFUSE(rows(a->dq, B, a->q_len, a->heads, true, "dq", &l.dq));
    H3_REFUSE(rows(a->dk, B, a->kv_len, a->kv_heads, true, "dk", &l.dk));
    H3_REFUSE(rows(a->dv, B, a->kv_len, a->kv_heads, true, "dv", &l.dv));
  }
  l.scale = a->scale;
  l.kv_lens = a->kv_lens;
  l.lse = a->lse;
  *L = l;
  return {};
}

Refusal check_workspace(const void* ws, size_t have, size_t need) {
  if (need == 0) return {};
  if (!ws || have < need)
    return no(H3C_ERR_CAPACITY, "needs " + std::to_string(need) + " bytes of workspace, has " +
                                    std::to_string(ws ? have : 0));
  if ((uintptr_t)ws & 255) return no(H3C_ERR_UNSUPPORTED, "workspace needs 256-byte alignment");
  return {};
}

size_t cross_workspace(const h3::CrossShape& n, int op) {
  return op == H3C_OP_CROSS_BWD ? h3::cross_bwd_workspace(n) : h3::cross_fwd_workspace(n);
}

h3c_status told(const Refusal& r, const char* who, char* err, size_t err_len) {
  if (err && err_len) std::snprintf(err, err_len, "%s%s%s", r ? who : "", r ? ": " : "", r.why.c_str());
  return r.status;
}

h3c_status cross_call(h3c_ctx* ctx, const h3c_cross_args* args, int op, const char* who, void* stream) try {
  if (!ctx) return H3C_ERR_INVALID_ARGUMENT;
  h3::CrossLaunch L;
  Refusal r = check_cross(args, op, &L);
  if (!r) r = check_workspace(args->workspace, args->workspace_bytes, cross_workspace(L.n, op));
  if (r) {
    ctx->err = std::string(who) + ": " + r.why;
    return r.status;
  }
  if (L.n.batch == 0) return H3C_OK;
  DeviceGuard guard(ctx->device);
  H3_CUDA_TRY(ctx, guard.err);
  L.ws = (uint8_t*)args->workspace;
  L.status = (int32_t*)(ctx->d_counter + 3);
  L.wait_limit_ns = h3::kWaitLimitNs;
  L.stall = -1;
  // Test hooks (fault injection on the host side): a shorter bound, as that of
  // h3c_attn_fwd, and beside it a barrier that waits for bytes that never come.
  if (const char* w = getenv("H3C_TEST_WAIT_LIMIT_NS")) {
    L.wait_limit_ns = strtoull(w, nullptr, 10);
    if (const char* b = getenv("H3C_TEST_STALL_BARRIER")) L.stall = atoi(b);
  }
  std::string why;
  cudaError_t e = op == H3C_OP_CROSS_BWD ? h3::launch_cross_bwd(L, (cudaStream_t)stream, &why)
                                         : h3::launch_cross_fwd(L, (cudaStream_t)stream, &why);
  if (e != cudaSuccess) {
    ctx->err = std::string(who) + ": " + why + cudaGetErrorString(e);
    return H3C_ERR_CUDA;
  }
  return H3C_OK;
} catch (const std::exception&) {
  return H3C_ERR_CAPACITY;  // host memory
}

Refusal check_norm(const h3c_qk_norm_args* a, bool bwd, h3::QkNormLaunch* L) {
  if (!a) return no(H3C_ERR_INVALID_ARGUMENT, "null args");
  if (a->head_dim != 128) return no(H3C_ERR_UNSUPPORTED, "head_dim must be 128");
  if (a->batch < 0 || a->q_len < 0 || a->k_len < 0 || a->heads <= 0 || a->kv_heads <= 0 || a->reserved != 0)
    return no(H3C_ERR_INVALID_ARGUMENT, "bad batch, lengths, heads or reserved");
  if (!(a->eps >= 0.f) || !std::isfinite(a->eps)) return no(H3C_ERR_INVALID_ARGUMENT, "eps must be finite and >= 0");
  if (!a->q_norm_weight || !a->k_norm_weight) return no(H3C_ERR_INVALID_ARGUMENT, "needs q/k norm weights");
  if (((uintptr_t)a->q_norm_weight & 15) || ((uintptr_t)a->k_norm_weight & 15) || ((uintptr_t)a->q_rope & 7) ||
      ((uintptr_t)a->k_rope & 7))
    return no(H3C_ERR_UNSUPPORTED, "norm weights need 16-byte, the rope tables 8-byte alignment");
  h3::QkNormLaunch l{};
  l.batch = a->batch;
  l.eps = a->eps;
  for (int i = 0; i < 2; ++i) {
    h3::QkNormOperand& o = l.op[i];
    o.tokens = i ? a->k_len : a->q_len;
    o.heads = i ? a->kv_heads : a->heads;
    o.w = (const uint16_t*)(i ? a->k_norm_weight : a->q_norm_weight);
    o.table = (const uint16_t*)(i ? a->k_rope : a->q_rope);
    o.half = o.table ? (i ? a->k_rope_half : a->q_rope_half) : 64;
    o.table_batch = i ? a->k_rope_batch_stride : a->q_rope_batch_stride;
    if (o.table && (o.half <= 0 || o.half > 64)) return no(H3C_ERR_UNSUPPORTED, "rope half must be in [1, 64]");
    if (o.table && a->batch > 1 && (o.table_batch < 0 || (o.table_batch & 3)))
      return no(H3C_ERR_INVALID_ARGUMENT, "a rope batch stride must be a multiple of 4 and not negative");
    if (product_over(a->batch, o.heads, o.tokens, INT_MAX - 65536)) return no(H3C_ERR_UNSUPPORTED, "more than 2^31 rows");
    const int64_t B = a->batch;
    H3_REFUSE(rows(i ? a->k : a->q, B, o.tokens, o.heads, false, i ? "k" : "q", &o.x));
    if (bwd) {
      o.dw = i ? a->k_norm_grad : a->q_norm_grad;
      if (!o.dw) return no(H3C_ERR_INVALID_ARGUMENT, "the backward call needs q_norm_grad and k_norm_grad");
      if ((uintptr_t)o.dw & 3) return no(H3C_ERR_UNSUPPORTED, "the norm gradients need 4-byte alignment");
      H3_REFUSE(rows(i ? a->k_grad : a->q_grad, B, o.tokens, o.heads, false, i ? "k_grad" : "q_grad", &o.g));
      H3_REFUSE(rows(i ? a->dk : a->dq, B, o.tokens, o.heads, true, i ? "dk" : "dq", &o.y));
    } else {
      H3_REFUSE(rows(i ? a->k_out : a->q_out, B, o.tokens, o.heads, true, i ? "k_out" : "q_out", &o.y));
    }
  }
  *L = l;
  return {};
}

h3c_status norm_call(h3c_ctx* ctx, const h3c_qk_norm_args* args, bool bwd, const char* who, void* stream) try {
  if (!ctx) return H3C_ERR_INVALID_ARGUMENT;
  h3::QkNormLaunch L;
  Refusal r = check_norm(args, bwd, &L);
  if (!r && bwd) r = check_workspace(args->workspace, args->workspace_bytes, h3::qk_norm_bwd_workspace());
  if (r) {
    ctx->err = std::string(who) + ": " + r.why;
    return r.status;
  }
  DeviceGuard guard(ctx->device);
  H3_CUDA_TRY(ctx, guard.err);
  L.ws = (float*)args->workspace;
  H3_CUDA_TRY(ctx, bwd ? h3::launch_qk_norm_bwd(L, (cudaStream_t)stream)
                       : h3::launch_qk_norm_fwd(L, (cudaStream_t)stream));
  return H3C_OK;
} catch (const std::exception&) {
  return H3C_ERR_CAPACITY;
}

}  // namespace

extern "C" {

h3c_status h3c_cross_workspace_size(const h3c_cross_args* args, int32_t op, size_t* bytes, char* err,
                                    size_t err_len) try {
  if (!bytes) return H3C_ERR_INVALID_ARGUMENT;
  *bytes = 0;
  h3::CrossLaunch L;
  Refusal r = check_cross(args, op, &L);
  if (!r) *bytes = cross_workspace(L.n, op);
  return told(r, "h3c_cross_workspace_size", err, err_len);
} catch (const std::exception&) {
  return H3C_ERR_CAPACITY;
}

h3c_status h3c_cross_attn_fwd(h3c_ctx* ctx, const h3c_cross_args* args, void* stream) {
  return cross_call(ctx, args, H3C_OP_CROSS_FWD, "h3c_cross_attn_fwd", stream);
}

h3c_status h3c_cross_attn_bwd(h3c_ctx* ctx, const h3c_cross_args* args, void* stream) {
  return cross_call(ctx, args, H3C_OP_CROSS_BWD, "h3c_cross_attn_bwd", stream);
}

h3c_status h3c_prefix_attn_fwd(h3c_ctx* ctx, const h3c_cross_args* args, void* stream) {
  return cross_call(ctx, args, H3C_OP_PREFIX_FWD, "h3c_prefix_attn_fwd", stream);
}

h3c_status h3c_qk_norm_workspace_size(const h3c_qk_norm_args* args, int32_t backward, size_t* bytes, char* err,
                                      size_t err_len) try {
  if (!bytes) return H3C_ERR_INVALID_ARGUMENT;
  *bytes = 0;
  h3::QkNormLaunch L;
  Refusal r = check_norm(args, backward != 0, &L);
  if (!r && backward) *bytes = h3::qk_norm_bwd_workspace();
  return told(r, "h3c_qk_norm_workspace_size", err, err_len);
} catch (const std::exception&) {
  return H3C_ERR_CAPACITY;
}

h3c_status h3c_qk_norm_rope_fwd(h3c_ctx* ctx, const h3c_qk_norm_args* args, void* stream) {
  return norm_call(ctx, args, false, "h3c_qk_norm_rope_fwd", stream);
}

h3c_status h3c_qk_norm_rope_bwd(h3c_ctx* ctx, const h3c_qk_norm_args* args, void* stream) {
  return norm_call(ctx, args, true, "h3c_qk_norm_rope_bwd", stream);
}

}  // extern "C"
