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
constexpr int MAX_DELTA_STRIDE = 1 << 24;  // of rows
constexpr uint64_t MAX_DELTA_STATES = 1ull << 36; // heads of all rays: a block each

int elem(int32_t dtype) { return dtype == FFN_F32 ? 4 : dtype == FFN_F16 || dtype == FFN_BF16 ? 2 : 0; }

bool aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }
bool words(const void* p) { return ((uintptr_t)p & 3) == 0; }  // of 4 bytes
bool aligned(const void* p, int64_t stride, int size) { return aligned(p) && stride * size % 16 == 0; }

// of two buffers of this many bytes
bool overlap(const void* p, const void* q, uint64_t bytes) {
  const uintptr_t x = (uintptr_t)p, y = (uintptr_t)q;
  return (x < y ? y - x : x - y) < bytes;
}

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

int check_plan(const int32_t* ids, uint32_t n, int32_t n_experts, const uint32_t* plan, uint64_t plan_words,
               const void* workspace, uint64_t workspace_bytes) {
  if (int rc = check_plan_sizes(n, n_experts)) return rc;
  if (n && !ids) return fail(-1, "NULL ids");
  const uint64_t words = ffn::expert_plan_words(n, n_experts), need = ffn::expert_plan_workspace(n, n_experts);
  if (!plan || !aligned(plan) || plan_words < words)
    return fail(-1, "plan of %llu words, %llu wanted", (unsigned long long)(plan ? plan_words : 0), (unsigned long long)words);
  if (need && (!workspace || !aligned(workspace) || workspace_bytes < need))
    return fail(-1, "workspace of %llu bytes, %llu wanted", (unsigned long long)(workspace ? workspace_bytes : 0),
                (unsigned long long)need);
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

int check_delta_sizes(const ffn_ray_delta* a) {
  if (!a) return fail(-1, "NULL arguments");
  if (!elem(a->dtype)) return fail(-1, "dtype=%d is not FFN_F32, FFN_F16 or FFN_BF16", a->dtype);
  if (a->heads < 1 || a->v_heads < 1 || a->v_heads > 1024 || a->v_heads % a->heads)
    return fail(-1, "v_heads=%d, heads=%d: v_heads must be a multiple of heads, at most 1024", a->v_heads, a->heads);
  if (a->key_dim < 8 || a->key_dim > 128 || a->key_dim % 8 || a->val_dim < 8 || a->val_dim > 128 || a->val_dim % 8)
    return fail(-1, "key_dim=%d, val_dim=%d must be multiples of 8, at most 128", a->key_dim, a->val_dim);
  if (a->reverse != 0 && a->reverse != 1) return fail(-1, "reverse=%d must be 0 or 1", a->reverse);
  if (a->rays.n > MAX_ROWS) return fail(-1, "rays: %u rows exceed %u", a->rays.n, MAX_ROWS);
  return 0;
}

int check_delta(const ffn_ray_delta* a, bool backward) {
  if (int rc = check_delta_sizes(a)) return rc;
  if (int rc = check_set(a->rays, "rays", true)) return rc;
  if (!(a->scale == a->scale) || a->scale > 3e38f || a->scale < -3e38f) return fail(-1, "scale=%g is not finite", a->scale);
  if ((uint64_t)a->rays.num_rays * a->v_heads > MAX_DELTA_STATES)
    return fail(-1, "%d heads of %u rays exceed 2^36", a->v_heads, a->rays.num_rays);
  const bool n = a->rays.n > 0;
  const int b = elem(a->dtype);
  const int64_t rows = a->rays.n, h = n ? a->heads : 0, vh = n ? a->v_heads : 0;
  if (n && (!a->q || !a->k || !a->v || !a->decay || !a->beta)) return fail(-1, "NULL buffer");
  const int64_t row_steps[] = {step(rows, a->q_row),    step(rows, a->k_row),    step(rows, a->v_row), step(rows, a->decay_row),
                               step(rows, a->beta_row), backward ? step(rows, a->do_row) : 0};
  for (int64_t s : row_steps)  // the kernels step through a chunk's rows with products of 24 bits
    if (s < 0 || s >= MAX_DELTA_STRIDE / b) return fail(-1, "row strides must be 0 or more, below %d bytes", MAX_DELTA_STRIDE);
  const int64_t head_steps[] = {step(h, a->q_head),      step(h, a->k_head),     step(vh, a->v_head), step(vh, a->decay_head),
                                step(vh, a->beta_head), backward ? step(vh, a->do_head) : 0};
  for (int64_t s : head_steps)
    if (s < 0) return fail(-1, "head strides must be 0 or more");
  if (!aligned(a->q, step(rows, a->q_row), b) || !aligned(a->q, step(h, a->q_head), b) || !aligned(a->k, step(rows, a->k_row), b) ||
      !aligned(a->k, step(h, a->k_head), b) || !aligned(a->v, step(rows, a->v_row), b) || !aligned(a->v, step(vh, a->v_head), b))
    return fail(-1, "rows and heads of q, k and v must be 16-byte aligned");
  if (((uintptr_t)a->decay | (uintptr_t)a->beta) & (b - 1)) return fail(-1, "misaligned decay or beta");
  if (!aligned(a->h0)) return fail(-1, "h0 must be 16-byte aligned");
  if (!backward) {
    if (n && !a->o) return fail(-1, "NULL output");
    if (!aligned(a->o) || !aligned(a->last) || !aligned(a->marks)) return fail(-1, "o, last and marks must be 16-byte aligned");
    const uint64_t states = (uint64_t)a->rays.num_rays * a->v_heads * a->key_dim * a->val_dim * sizeof(float);
    if (a->h0 && a->last && states) {
      if (a->last == a->h0) {
        if (a->marks) return fail(-1, "last is h0, and marks are asked for: the backward reads h0");
      } else if (overlap(a->last, a->h0, states)) {
        return fail(-1, "last overlaps h0 without being it");
      }
    }
    return 0;
  }
  if (n && (!a->dout || !a->dq || !a->dk || !a->dv || !a->ddecay || !a->dbeta || !a->marks))
    return fail(-1, "NULL gradient buffer or marks");
  if (!aligned(a->dout, step(rows, a->do_row), b) || !aligned(a->dout, step(vh, a->do_head), b) || !aligned(a->dq) ||
      !aligned(a->dk) || !aligned(a->dv) || !aligned(a->ddecay) || !aligned(a->dbeta) || !aligned(a->dlast) || !aligned(a->dh0) ||
      !aligned(a->marks))
    return fail(-1, "rows and heads of the gradients, the states' gradients and marks must be 16-byte aligned");
  const uint64_t need = ffn::delta_workspace(*a);
  if (need && (!a->workspace || !aligned(a->workspace) || a->workspace_bytes < need))
    return fail(-1, "workspace of %llu bytes, %llu wanted", (unsigned long long)(a->workspace ? a->workspace_bytes : 0),
                (unsigned long long)need);
  return 0;
}

int check_norm(const ffn_norm* a) {
  if (!a) return fail(-1, "NULL arguments");
  if (!elem(a->dtype)) return fail(-1, "dtype=%d is not FFN_F32, FFN_F16 or FFN_BF16", a->dtype);
  if (a->param_dtype != FFN_F32 && a->param_dtype != a->dtype)
    return fail(-1, "param_dtype=%d must be FFN_F32 or dtype=%d", a->param_dtype, a->dtype);
  if (a->width < 1 || a->width > FFN_NORM_MAX_WIDTH)
    return fail(-1, "width=%d must be 1 to %d", a->width, FFN_NORM_MAX_WIDTH);
  if (a->n > MAX_ROWS) return fail(-1, "%u rows exceed %u", a->n, MAX_ROWS);
  if (!(a->eps >= 0.f) || a->eps > 3e38f) return fail(-1, "eps=%g must be 0 or positive", a->eps);
  const uintptr_t odd = elem(a->dtype) - 1, podd = elem(a->param_dtype) - 1;
  if (((uintptr_t)a->x | (uintptr_t)a->y | (uintptr_t)a->dy | (uintptr_t)a->dx) & odd) return fail(-1, "misaligned buffer");
  if (((uintptr_t)a->weight | (uintptr_t)a->bias) & podd) return fail(-1, "misaligned parameters");
  if (!words(a->mean) || !words(a->rstd) || !words(a->dweight) || !words(a->dbias))
    return fail(-1, "misaligned mean, rstd, dweight or dbias");
  return 0;
}

int check_route(const ffn_route* a) {
  if (!a) return fail(-1, "NULL arguments");
  if (!elem(a->dtype)) return fail(-1, "dtype=%d is not FFN_F32, FFN_F16 or FFN_BF16", a->dtype);
  if (a->k < 1 || a->k > FFN_MAX_EXPERTS) return fail(-1, "k=%d must be 1 to %d", a->k, FFN_MAX_EXPERTS);
  if (a->width < 1 || a->width > 65536) return fail(-1, "width=%d must be 1 to 65536", a->width);
  const uint64_t places = (uint64_t)a->n * a->k;
  if (places > MAX_ROWS) return fail(-1, "%llu places exceed %u", (unsigned long long)places, MAX_ROWS);
  if (int rc = check_plan_sizes((uint32_t)places, a->n_experts)) return rc;
  if (a->n && (!a->plan || !a->slots)) return fail(-1, "NULL plan or slots");
  if (a->rows_stride < 0 || a->slots_stride < 0) return fail(-1, "row strides must be 0 or more");
  const uintptr_t odd = elem(a->dtype) - 1;
  if (((uintptr_t)a->rows_in | (uintptr_t)a->slots_in | (uintptr_t)a->rows_out | (uintptr_t)a->slots_out) & odd)
    return fail(-1, "misaligned buffer");
  if (!words(a->plan) || !words(a->slots) || !words(a->weights) || !words(a->dweights))
    return fail(-1, "misaligned plan, slots, weights or dweights");
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

int ffn_ray_delta_marks(const ffn_ray_delta* a, uint64_t* bytes) {
  if (int rc = check_delta_sizes(a)) return rc;
  if (!bytes) return fail(-1, "NULL bytes");
  *bytes = ffn::delta_marks(*a);
  return 0;
}

int ffn_ray_delta_workspace(const ffn_ray_delta* a, int32_t backward, uint64_t* bytes) {
  if (int rc = check_delta_sizes(a)) return rc;
  if (!bytes) return fail(-1, "NULL bytes");
  *bytes = backward ? ffn::delta_workspace(*a) : 0;
  return 0;
}

int ffn_ray_delta_fwd(const ffn_ray_delta* a, void* stream) {
  if (int rc = check_delta(a, false)) return rc;
  return launched(ffn::launch_delta(*a, false, (hipStream_t)stream), "ffn_ray_delta_fwd");
}

int ffn_ray_delta_bwd(const ffn_ray_delta* a, void* stream) {
  if (int rc = check_delta(a, true)) return rc;
  return launched(ffn::launch_delta(*a, true, (hipStream_t)stream), "ffn_ray_delta_bwd");
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
  if (int rc = check_plan(ids, n, n_experts, plan, plan_words, workspace, workspace_bytes)) return rc;
  return launched(ffn::launch_expert_plan(ids, n, n_experts, plan, nullptr, (uint32_t*)workspace, (hipStream_t)stream),
                  "ffn_expert_plan");
}

int ffn_expert_route(const int32_t* ids, uint32_t places, int32_t n_experts, uint32_t* plan, uint64_t plan_words, uint32_t* slots,
                     void* workspace, uint64_t workspace_bytes, void* stream) {
  if (int rc = check_plan(ids, places, n_experts, plan, plan_words, workspace, workspace_bytes)) return rc;
  if (places && !slots) return fail(-1, "NULL slots");
  if (!words(ids) || !words(slots)) return fail(-1, "misaligned ids or slots");
  return launched(ffn::launch_expert_plan(ids, places, n_experts, plan, slots, (uint32_t*)workspace, (hipStream_t)stream),
                  "ffn_expert_route");
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

int ffn_layer_norm_fwd(const ffn_norm* a, void* stream) {
  if (int rc = check_norm(a)) return rc;
  if (a->n == 0) return 0;
  if (!a->x || !a->y || !a->mean || !a->rstd) return fail(-1, "NULL buffer");
  return launched(ffn::launch_norm(*a, false, (hipStream_t)stream), "ffn_layer_norm_fwd");
}

int ffn_layer_norm_workspace(const ffn_norm* a, uint64_t* bytes) {
  if (int rc = check_norm(a)) return rc;
  if (!bytes) return fail(-1, "NULL bytes");
  *bytes = ffn::norm_workspace(*a);
  return 0;
}

int ffn_layer_norm_bwd(const ffn_norm* a, void* stream) {
  if (int rc = check_norm(a)) return rc;
  if (a->n && (!a->x || !a->dy || !a->mean || !a->rstd)) return fail(-1, "NULL buffer");
  const uint64_t need = a->dweight || a->dbias ? ffn::norm_workspace(*a) : 0;
  if (need && (!a->workspace || !aligned(a->workspace) || a->workspace_bytes < need))
    return fail(-1, "workspace of %llu bytes, %llu wanted", (unsigned long long)(a->workspace ? a->workspace_bytes : 0),
                (unsigned long long)need);
  return launched(ffn::launch_norm(*a, true, (hipStream_t)stream), "ffn_layer_norm_bwd");
}

int ffn_expert_dispatch(const ffn_route* a, void* stream) {
  if (int rc = check_route(a)) return rc;
  if (a->n && (!a->rows_in || !a->slots_out)) return fail(-1, "NULL buffer");
  return launched(ffn::launch_dispatch(*a, (hipStream_t)stream), "ffn_expert_dispatch");
}

int ffn_expert_combine(const ffn_route* a, void* stream) {
  if (int rc = check_route(a)) return rc;
  if (a->n && (!a->slots_in || !a->rows_out)) return fail(-1, "NULL buffer");
  return launched(ffn::launch_combine(*a, (hipStream_t)stream), "ffn_expert_combine");
}

int ffn_expert_combine_bwd(const ffn_route* a, void* stream) {
  if (int rc = check_route(a)) return rc;
  if (a->n && (!a->rows_in || !a->slots_out || (a->dweights && !a->slots_in))) return fail(-1, "NULL buffer");
  return launched(ffn::launch_combine_bwd(*a, (hipStream_t)stream), "ffn_expert_combine_bwd");
}

}  // extern "C"
