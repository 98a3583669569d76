// ffn_ray_capi.hip -- the C entry points of the operators along rays and of the expert layers
// (include/ffnerf_hip.h): they check their arguments, and launch.
#include <stdarg.h>
#include <stdio.h>

#include "ffn_ray_kernels.h"

namespace {

int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return ffn::set_error(code, buf);
}

int launched(hipError_t e, const char* what) {
  return e == hipSuccess ? 0 : fail(-3, "%s: %s", what, hipGetErrorString(e));
}

// row numbers are 32-bit with room for a tile past the end
constexpr uint32_t MAX_ROWS = 0x7FFFFF00u;

constexpr int MAX_SCAN_STRIDE = 1 << 27;

constexpr uint64_t MAX_SCAN_STATES = 1ull << 46;  // channels of all rays: what one launch can count

int elem(int32_t dtype) { return dtype == FFN_F32 ? 4 : dtype == FFN_F16 || dtype == FFN_BF16 ? 2 : 0; }

bool aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }
bool aligned(const void* p, int64_t stride, int size) { return aligned(p) && stride * size % 16 == 0; }

// the stride of an axis of `count`: that of one place, or none, is any number and leads nowhere
int64_t step(int64_t count, int64_t stride) { return count > 1 ? stride : 0; }

int check_set(const ffn_ray_set& s, const char* name, bool ids) {
  if (s.n > MAX_ROWS) return fail(-1, "%s: %u rows exceed %u", name, s.n, MAX_ROWS);
  if (s.num_rays && (!s.counts || !s.offsets)) return fail(-1, "%s: NULL counts or offsets", name);
  if (ids && s.n && !s.ray_ids) return fail(-1, "%s: NULL ray_ids", name);
  return 0;
}

int check_sizes(const ffn_ray_attn* a) {
  if (!a) return fail(-1, "NULL arguments");
  if (!elem(a->dtype)) return fail(-1, "dtype=%d is not FFN_F32, FFN_F16 or FFN_BF16", a->dtype);
  if (a->heads < 1 || a->kv_heads < 1 || a->heads > 1024 || a->heads % a->kv_heads)
    return fail(-1, "heads=%d, kv_heads=%d: heads must be a multiple of kv_heads, at most 1024", a->heads, a->kv_heads);
  if (a->dim < 8 || a->dim > 128 || a->dim % 8) return fail(-1, "dim=%d must be a multiple of 8, at most 128", a->dim);
  if (a->q_rays.num_rays != a->k_rays.num_rays)
    return fail(-1, "queries of %u rays, keys of %u", a->q_rays.num_rays, a->k_rays.num_rays);
  return 0;
}

int check_attn(const ffn_ray_attn* a, bool backward) {
  if (int rc = check_sizes(a)) return rc;
  if (int rc = check_set(a->q_rays, "q_rays", true)) return rc;
  if (int rc = check_set(a->k_rays, "k_rays", backward)) return rc;
  if (!(a->cap >= 0.f) || a->cap > 3e38f) return fail(-1, "cap=%g must be 0 (none) or positive", a->cap);
  if (!(a->scale == a->scale) || a->scale > 3e38f || a->scale < -3e38f) return fail(-1, "scale=%g is not finite", a->scale);
  const int b = elem(a->dtype);
  const bool nq = a->q_rays.n > 0, nk = a->k_rays.n > 0;
  if ((nq && (!a->q || !a->o || !a->lse)) || (nk && (!a->k || !a->v))) return fail(-1, "NULL buffer");
  const int64_t qn = a->q_rays.n, kn = a->k_rays.n, qh = nq ? a->heads : 0, kh = nk ? a->kv_heads : 0;
  if (!aligned(a->q, step(qn, a->q_row), b) || !aligned(a->q, step(qh, a->q_head), b) ||
      !aligned(a->k, step(kn, a->k_row), b) || !aligned(a->k, step(kh, a->k_head), b) ||
      !aligned(a->v, step(kn, a->v_row), b) || !aligned(a->v, step(kh, a->v_head), b) || !aligned(a->o))
    return fail(-1, "rows and heads of q, k, v and o must be 16-byte aligned");
  if (a->slopes && ((nq && !a->t_q) || (nk && !a->t_k))) return fail(-1, "slopes without t_q and t_k");
  if (backward) {
    if ((nq && (!a->dout || !a->dq)) || (nk && (!a->dk || !a->dv))) return fail(-1, "NULL gradient buffer");
    if (!aligned(a->dout, step(qn, a->do_row), b) || !aligned(a->dout, step(qh, a->do_head), b) || !aligned(a->dq) ||
        !aligned(a->dk) || !aligned(a->dv))
      return fail(-1, "rows and heads of the gradients must be 16-byte aligned");
  }
  const uint64_t need = ffn::attn_workspace(*a, backward);
  if (need && (!a->workspace || !aligned(a->workspace) || a->workspace_bytes < need))
    return fail(-1, "workspace of %llu bytes, %llu wanted", (unsigned long long)(a->workspace ? a->workspace_bytes : 0),
                (unsigned long long)need);
  return 0;
}

int check_scan_sizes(const ffn_ray_scan* a) {
  if (!a) return fail(-1, "NULL arguments");
  if (!elem(a->dtype)) return fail(-1, "dtype=%d is not FFN_F32, FFN_F16 or FFN_BF16", a->dtype);
  if (a->channels < 1 || a->channels > 65536) return fail(-1, "channels=%d must be 1 to 65536", a->channels);
  if (a->reverse != 0 && a->reverse != 1) return fail(-1, "reverse=%d must be 0 or 1", a->reverse);
  return 0;
}

int check_scan(const ffn_ray_scan* a, bool backward) {
  if (int rc = check_scan_sizes(a)) return rc;
  if (int rc = check_set(a->rays, "rays", true)) return rc;
  const bool n = a->rays.n > 0;
  const uintptr_t odd = elem(a->dtype) - 1;
  if (n && (!a->gate || !a->x)) return fail(-1, "NULL buffer");
  if (n && !backward && !a->h) return fail(-1, "NULL output");
  if (n && backward && (!a->dh || !a->dgate || !a->dx || !a->marks)) return fail(-1, "NULL gradient buffer or marks");
  if (((uintptr_t)a->gate | (uintptr_t)a->x | (uintptr_t)a->h) & odd) return fail(-1, "misaligned buffer");
  if (backward && ((uintptr_t)a->dh | (uintptr_t)a->dgate | (uintptr_t)a->dx) & odd)
    return fail(-1, "misaligned gradient buffer");
  // the kernels step through a few rows with 32-bit offsets
  const int64_t far = (int64_t)MAX_SCAN_STRIDE / elem(a->dtype);
  if (a->rays.n > 1 && (a->gate_row > far || a->gate_row < -far || a->x_row > far || a->x_row < -far ||
                        (backward && (a->dh_row > far || a->dh_row < -far))))
    return fail(-1, "rows more than %d bytes apart", MAX_SCAN_STRIDE);
  if ((uint64_t)a->rays.num_rays * a->channels > MAX_SCAN_STATES)
    return fail(-1, "%d channels of %u rays exceed 2^46", a->channels, a->rays.num_rays);
  const uint64_t need = ffn::scan_workspace(*a, backward);
  if (need && (!a->workspace || !aligned(a->workspace) || a->workspace_bytes < need))
    return fail(-1, "workspace of %llu bytes, %llu wanted", (unsigned long long)(a->workspace ? a->workspace_bytes : 0),
                (unsigned long long)need);
  return 0;
}

int check_plan_sizes(uint32_t n, int32_t n_experts) {
  if (n > MAX_ROWS) return fail(-1, "%u rows exceed %u", n, MAX_ROWS);
  if (n_experts < 1 || n_experts > FFN_MAX_EXPERTS)
    return fail(-1, "n_experts=%d must be 1 to %d", n_experts, FFN_MAX_EXPERTS);
  return 0;
}

int check_experts(const ffn_experts* a) {
  if (!a) return fail(-1, "NULL arguments");
  if (!elem(a->dtype)) return fail(-1, "dtype=%d is not FFN_F32, FFN_F16 or FFN_BF16", a->dtype);
  if (int rc = check_plan_sizes(a->n, a->n_experts)) return rc;
  if (a->in < 8 || a->in > 4096 || a->in % 8 || a->out < 8 || a->out > 4096 || a->out % 8)
    return fail(-1, "in=%d, out=%d must be multiples of 8, at most 4096", a->in, a->out);
  if (a->flags & ~(FFN_EXPERTS_X_SLOTS | FFN_EXPERTS_Y_SLOTS)) return fail(-1, "unknown flags %d", a->flags);
  if (!a->plan) return fail(-1, "NULL plan");
  const int64_t far = (int64_t)(UINT32_MAX / elem(a->dtype));
  if (a->n > 1 && (a->x_row < 0 || a->x_row > far || a->dy_row < 0 || a->dy_row > far))
    return fail(-1, "row strides must be 0 or more, and less than 4 GiB");
  return 0;
}

}  // namespace

extern "C" {

int ffn_ray_attention_workspace(const ffn_ray_attn* a, int32_t backward, uint64_t* bytes) {
  if (int rc = check_sizes(a)) return rc;
  if (!bytes) return fail(-1, "NULL bytes");
  *bytes = ffn::attn_workspace(*a, backward != 0);
  return 0;
}

int ffn_ray_attention_fwd(const ffn_ray_attn* a, void* stream) {
  if (int rc = check_attn(a, false)) return rc;
  if (a->q_rays.n == 0) return 0;
  return launched(ffn::launch_attn(*a, false, (hipStream_t)stream), "ffn_ray_attention_fwd");
}

int ffn_ray_attention_bwd(const ffn_ray_attn* a, void* stream) {
  if (int rc = check_attn(a, true)) return rc;
  return launched(ffn::launch_attn(*a, true, (hipStream_t)stream), "ffn_ray_attention_bwd");
}

int ffn_ray_scan_marks(const ffn_ray_scan* a, uint64_t* bytes) {
  if (int rc = check_scan_sizes(a)) return rc;
  if (!bytes) return fail(-1, "NULL bytes");
  *bytes = ffn::scan_marks(*a);
  return 0;
}

int ffn_ray_scan_workspace(const ffn_ray_scan* a, int32_t backward, uint64_t* bytes) {
  if (int rc = check_scan_sizes(a)) return rc;
  if (!bytes) return fail(-1, "NULL bytes");
  *bytes = ffn::scan_workspace(*a, backward != 0);
  return 0;
}

int ffn_ray_scan_fwd(const ffn_ray_scan* a, void* stream) {
  if (int rc = check_scan(a, false)) return rc;
  return launched(ffn::launch_scan(*a, false, (hipStream_t)stream), "ffn_ray_scan_fwd");
}

int ffn_ray_scan_bwd(const ffn_ray_scan* a, void* stream) {
  if (int rc = check_scan(a, true)) return rc;
  return launched(ffn::launch_scan(*a, true, (hipStream_t)stream), "ffn_ray_scan_bwd");
}

int ffn_expert_plan_size(uint32_t n, int32_t n_experts, uint64_t* plan_words, uint64_t* workspace_bytes) {
  if (int rc = check_plan_sizes(n, n_experts)) return rc;
  if (!plan_words || !workspace_bytes) return fail(-1, "NULL result");
  *plan_words = ffn::expert_plan_words(n, n_experts);
  *workspace_bytes = ffn::expert_plan_workspace(n, n_experts);
  return 0;
}

int ffn_expert_plan(const int32_t* ids, uint32_t n, int32_t n_experts, uint32_t* plan, uint64_t plan_words,
                    void* workspace, uint64_t workspace_bytes, void* stream) {
  if (int rc = check_plan_sizes(n, n_experts)) return rc;
  if (n && !ids) return fail(-1, "NULL ids");
  const uint64_t words = ffn::expert_plan_words(n, n_experts), need = ffn::expert_plan_workspace(n, n_experts);
  if (!plan || !aligned(plan) || plan_words < words)
    return fail(-1, "plan of %llu words, %llu wanted", (unsigned long long)(plan ? plan_words : 0), (unsigned long long)words);
  if (need && (!workspace || !aligned(workspace) || workspace_bytes < need))
    return fail(-1, "workspace of %llu bytes, %llu wanted", (unsigned long long)(workspace ? workspace_bytes : 0),
                (unsigned long long)need);
  return launched(ffn::launch_expert_plan(ids, n, n_experts, plan, (uint32_t*)workspace, (hipStream_t)stream),
                  "ffn_expert_plan");
}

int ffn_expert_linear_fwd(const ffn_experts* a, void* stream) {
  if (int rc = check_experts(a)) return rc;
  const int b = elem(a->dtype);
  if (a->n == 0) return 0;
  if (!a->x || !a->W || !a->y) return fail(-1, "NULL buffer");
  if (!aligned(a->x, step(a->n, a->x_row), b) || !aligned(a->W) || !aligned(a->b) || !aligned(a->y))
    return fail(-1, "rows of x, W, b and y must be 16-byte aligned");
  return launched(ffn::launch_experts(*a, false, (hipStream_t)stream), "ffn_expert_linear_fwd");
}

int ffn_expert_linear_workspace(const ffn_experts* a, uint64_t* bytes) {
  if (int rc = check_experts(a)) return rc;
  if (!bytes) return fail(-1, "NULL bytes");
  *bytes = ffn::expert_workspace(*a);
  return 0;
}

int ffn_expert_linear_bwd(const ffn_experts* a, void* stream) {
  if (int rc = check_experts(a)) return rc;
  const int b = elem(a->dtype);
  if (a->n && (!a->dy || (a->relu && !a->y) || (a->dx && !a->W) || ((a->dW || a->db) && !a->x)))
    return fail(-1, "NULL buffer");
  if (!aligned(a->dy, step(a->n, a->dy_row), b) || !aligned(a->y) || !aligned(a->W) || !aligned(a->x, step(a->n, a->x_row), b) ||
      !aligned(a->dx) || !aligned(a->dW) || !aligned(a->db))
    return fail(-1, "rows of dy, y, W, x and the gradients must be 16-byte aligned");
  const uint64_t need = ffn::expert_workspace(*a);
  if (need && (!a->workspace || !aligned(a->workspace) || a->workspace_bytes < need))
    return fail(-1, "workspace of %llu bytes, %llu wanted", (unsigned long long)(a->workspace ? a->workspace_bytes : 0),
                (unsigned long long)need);
  return launched(ffn::launch_experts(*a, true, (hipStream_t)stream), "ffn_expert_linear_bwd");
}

}  // extern "C"
