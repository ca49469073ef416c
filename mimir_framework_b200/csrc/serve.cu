// serve.cu — the C calls of the serving group: what the host can see of their arguments is checked here, what lies in device memory by
// the kernels (paged.cuh).
#include <cmath>

#include "common.h"
#include "host_call.h"
#include "layer.cuh"
#include "paged.cuh"

namespace mb {

// words[2] = words[1], which is left at zero, in one step: what another stream finds meanwhile is in the one or in the other
__global__ void take_findings_kernel(int* words) { words[2] = atomicExch(words + 1, 0); }

int paged_flags_read(cudaStream_t st) {
  Context& c = ctx();
  if (!c.paged_used.load()) return MIMIR_B200_OK;
  int flags = 0;
  auto look = [&](int word) -> int {
    MB_CUDA(cudaMemcpyAsync(&flags, c.dev_error_word + word, sizeof(int), cudaMemcpyDeviceToHost, st));
    MB_CUDA(cudaStreamSynchronize(st));
    return MIMIR_B200_OK;
  };
  MB_TRY(look(1));
  if (!flags) return MIMIR_B200_OK;
  {
    std::lock_guard<std::mutex> lk(c.error_mu);  // (words[2] is one call's at a time)
    take_findings_kernel<<<1, 1, 0, st>>>(c.dev_error_word);
    MB_CUDA(cudaGetLastError());
    count_launch();
    MB_TRY(look(2));
  }
  if (!flags) return MIMIR_B200_OK;  // (another thread has them)
  return fail(MIMIR_B200_E_INVALID, "paged batch:%s%s%s", (flags & PAGED_BAD_ROWS) ? " row ranges that do not fit the tensors;" : "",
              (flags & PAGED_BAD_LEN) ? " a key count that does not fit max_kv or the page table;" : "",
              (flags & PAGED_BAD_PAGE) ? " a page number outside the cache;" : "");
}

namespace {

bool row_type(int t) { return t == MIMIR_B200_T_F32 || t == MIMIR_B200_T_F16 || t == MIMIR_B200_T_BF16; }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Device memory, as far as the driver can tell (a pointer it has never seen is the host's).
int check_device_pointer(const char* what, const char* name, const void* p) {
  if (!p) return fail(MIMIR_B200_E_INVALID, "%s: %s is null", what, name);
  cudaPointerAttributes at;
  if (cudaPointerGetAttributes(&at, p) != cudaSuccess) {
    cudaGetLastError();
    return fail(MIMIR_B200_E_INVALID, "%s: %s is not a device pointer", what, name);
  }
  if (at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged) return fail(MIMIR_B200_E_INVALID, "%s: %s is not a device pointer", what, name);
  if (at.type == cudaMemoryTypeDevice && at.device != ctx().device)
    return fail(MIMIR_B200_E_INVALID, "%s: %s is on device %d, the current device is %d", what, name, at.device, ctx().device);
  return MIMIR_B200_OK;
}
// ... of 4-byte words
int check_device_words(const char* what, const char* name, const void* p) {
  MB_TRY(check_device_pointer(what, name, p));
  if (reinterpret_cast<uintptr_t>(p) & 3) return fail(MIMIR_B200_E_INVALID, "%s: %s is not 4-byte aligned", what, name);
  return MIMIR_B200_OK;
}

// the sizes of a cache and a batch (no pointers)
int check_sizes(const char* what, const MimirPagedCache* c, const MimirPagedBatch* b) {
  if (!c || !b) return fail(MIMIR_B200_E_INVALID, "%s: null argument", what);
  if (c->type < MIMIR_B200_T_F32 || c->type > MIMIR_B200_T_E4M3) return fail(MIMIR_B200_E_INVALID, "%s: unknown cache type %d", what, c->type);
  if (c->n_pages <= 0 || c->kv_heads <= 0 || c->page_size <= 0 || c->head_dim <= 0)
    return fail(MIMIR_B200_E_INVALID, "%s: the cache has no pages, slots, heads or elements", what);
  if (c->page_size % 8) return fail(MIMIR_B200_E_UNSUPPORTED, "%s: page_size %d is not a multiple of 8", what, c->page_size);
  if (c->head_dim % 8 || c->head_dim > 256) return fail(MIMIR_B200_E_UNSUPPORTED, "%s: head_dim %d is not a multiple of 8 up to 256", what, c->head_dim);
  if (c->page_stride % 8 || c->slot_stride % 8 || c->head_stride % 8 || c->page_stride < 0 || c->slot_stride < 0 || c->head_stride < 0)
    return fail(MIMIR_B200_E_UNSUPPORTED, "%s: cache strides are multiples of 8 elements", what);
  if ((c->page_size > 1 && c->slot_stride == 0) || (c->kv_heads > 1 && c->head_stride == 0) || (c->n_pages > 1 && c->page_stride == 0) ||
      c->page_stride >= (1LL << 38) || c->slot_stride >= (1LL << 38) || c->head_stride >= (1LL << 38))
    return fail(MIMIR_B200_E_UNSUPPORTED, "%s: cache strides are positive and below 2^38 elements", what);
  if (b->n_seqs < 0 || b->n_rows < 0 || b->max_rows < 0 || b->max_kv < 0 || b->table_stride < 0)
    return fail(MIMIR_B200_E_INVALID, "%s: a negative size in the batch", what);
  return MIMIR_B200_OK;
}

int check_pointers(const char* what, const MimirPagedCache* c, const MimirPagedBatch* b, PagedView* v, bool rows) {
  MB_TRY(check_device_pointer(what, "the cache's k", c->k));
  MB_TRY(check_device_pointer(what, "the cache's v", c->v));
  const bool coded = c->type == MIMIR_B200_T_I8 || c->type == MIMIR_B200_T_E4M3;
  if (coded) {
    MB_TRY(check_device_words(what, "the cache's k_scale", c->k_scale));
    MB_TRY(check_device_words(what, "the cache's v_scale", c->v_scale));
  }
  if (!aligned16(c->k) || !aligned16(c->v) || (coded && (!aligned16(c->k_scale) || !aligned16(c->v_scale))))
    return fail(MIMIR_B200_E_UNSUPPORTED, "%s: the cache's pointers are not 16-byte aligned", what);
  if (rows) MB_TRY(check_device_words(what, "row_start", b->row_start));
  MB_TRY(check_device_words(what, "kv_len", b->kv_len));
  if (b->table_stride > 0) MB_TRY(check_device_words(what, "page_table", b->page_table));
  v->k = c->k, v->v = c->v, v->k_scale = c->k_scale, v->v_scale = c->v_scale;
  v->page_stride = c->page_stride, v->slot_stride = c->slot_stride, v->head_stride = c->head_stride;
  v->n_pages = c->n_pages, v->page_size = c->page_size, v->kv_heads = c->kv_heads, v->head_dim = c->head_dim;
  v->by_page = FastDiv(static_cast<uint32_t>(c->page_size));
  v->row_start = b->row_start, v->kv_len = b->kv_len, v->table = b->page_table, v->table_stride = b->table_stride;
  v->n_seqs = b->n_seqs, v->n_rows = b->n_rows, v->max_rows = b->max_rows, v->max_kv = b->max_kv;
  v->flags = ctx().dev_error_word + 1;
  ctx().paged_used.store(true);
  return MIMIR_B200_OK;
}

int check_row_tensors(const char* what, const void* a, const void* b, int type, long long row_stride, long long head_stride) {
  if (!row_type(type)) return fail(MIMIR_B200_E_INVALID, "%s: rows are F32, F16 or BF16, not type %d", what, type);
  MB_TRY(check_device_pointer(what, "k", a));
  MB_TRY(check_device_pointer(what, "v", b));
  if (row_stride % 8 || head_stride % 8 || row_stride < 0 || head_stride < 0 || !aligned16(a) || !aligned16(b))
    return fail(MIMIR_B200_E_UNSUPPORTED, "%s: row tensors start on 16 bytes and have strides of multiples of 8 elements", what);
  return MIMIR_B200_OK;
}

int check_attention(const char* what, const MimirPagedCache* c, const MimirPagedBatch* b, const MimirPagedAttention* at, AttendLaunch* l) {
  MB_TRY(check_sizes(what, c, b));
  if (!at) return fail(MIMIR_B200_E_INVALID, "%s: null argument", what);
  if (!row_type(at->type)) return fail(MIMIR_B200_E_INVALID, "%s: q and out are F32, F16 or BF16, not type %d", what, at->type);
  if (at->heads <= 0 || at->heads % c->kv_heads) return fail(MIMIR_B200_E_INVALID, "%s: %d heads are no multiple of %d key heads", what, at->heads, c->kv_heads);
  if (at->window < 0) return fail(MIMIR_B200_E_INVALID, "%s: negative window", what);
  if (!std::isfinite(at->scale)) return fail(MIMIR_B200_E_INVALID, "%s: the scale is not finite", what);
  if ((c->type == MIMIR_B200_T_F32 && at->type != MIMIR_B200_T_F32) || (c->type == MIMIR_B200_T_BF16 && at->type != MIMIR_B200_T_BF16))
    return fail(MIMIR_B200_E_UNSUPPORTED, "%s: a cache of type F32 or BF16 takes queries of its own type", what);
  if (at->row_stride % 8 || at->head_stride % 8 || at->out_row_stride % 8 || at->out_head_stride % 8 || at->row_stride < 0 || at->head_stride < 0 ||
      at->out_row_stride < 0 || at->out_head_stride < 0)
    return fail(MIMIR_B200_E_UNSUPPORTED, "%s: strides of q and out are multiples of 8 elements", what);
  l->p.n_seqs = b->n_seqs, l->p.n_rows = b->n_rows, l->p.max_rows = b->max_rows < b->n_rows ? b->max_rows : b->n_rows, l->p.max_kv = b->max_kv;
  l->p.kv_heads = c->kv_heads, l->p.head_dim = c->head_dim, l->p.page_size = c->page_size;
  if (static_cast<long long>(l->p.max_rows) * at->heads > 0x7fffffffLL) return fail(MIMIR_B200_E_INVALID, "%s: too many rows and heads for one call", what);
  if (l->p.max_kv > (1 << 30)) l->p.max_kv = 1 << 30;  // (key numbers leave room to round up; a longer sequence is reported as one that does not fit)
  // a window that no sequence fills is none
  l->cache_type = c->type, l->type = at->type, l->heads = at->heads, l->causal = at->causal != 0, l->scale = at->scale;
  l->window = at->window < l->p.max_kv ? at->window : 0;
  l->q = at->q, l->out = at->out, l->lse = at->lse, l->ws = at->workspace, l->ws_bytes = at->workspace_bytes;
  l->q_row = at->row_stride, l->q_head = at->head_stride, l->o_row = at->out_row_stride, l->o_head = at->out_head_stride;
  return MIMIR_B200_OK;
}

// ---- a layer's norms and products ---------------------------------------------------------------------------------------------------
bool on_boundary(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % static_cast<uintptr_t>(bytes) == 0; }
// rows of `wide` elements, `stride` apart, that do not run into one another
int check_row_stride(const char* what, const char* name, long long stride, long long rows, long long wide) {
  if (stride < 0 || (rows > 1 && stride < wide) || stride >= (1LL << 36))
    return fail(MIMIR_B200_E_INVALID, "%s: %s has rows of %lld elements, %lld apart", what, name, wide, stride);
  return MIMIR_B200_OK;
}

int check_norm_rows(const MimirNormRows* a) {
  const char* what = "norm_rows";
  if (!a) return fail(MIMIR_B200_E_INVALID, "%s: null argument", what);
  if (!row_type(a->type)) return fail(MIMIR_B200_E_INVALID, "%s: x is F32, F16 or BF16, not type %d", what, a->type);
  if (!row_type(a->y_type) && a->y_type != MIMIR_B200_T_E4M3)
    return fail(a->y_type == MIMIR_B200_T_I8 ? MIMIR_B200_E_UNSUPPORTED : MIMIR_B200_E_INVALID, "%s: y is F32, F16, BF16 or E4M3, not type %d", what, a->y_type);
  if (a->rows < 0 || a->n <= 0) return fail(MIMIR_B200_E_INVALID, "%s: %d rows of %d", what, a->rows, a->n);
  if (a->n > 32768) return fail(MIMIR_B200_E_UNSUPPORTED, "%s: rows of %d elements (32 768 at most)", what, a->n);
  if (a->norm && !(a->eps >= 0.0f && std::isfinite(a->eps))) return fail(MIMIR_B200_E_INVALID, "%s: eps is negative or not finite", what);
  if (!a->norm && a->gamma) return fail(MIMIR_B200_E_INVALID, "%s: gamma without the norm", what);
  if ((a->y_type == MIMIR_B200_T_E4M3) != (a->y_scale != nullptr)) return fail(MIMIR_B200_E_INVALID, "%s: y_scale belongs to a y of type E4M3", what);
  MB_TRY(check_row_stride(what, "x", a->x_stride, a->rows, a->n));
  if (a->residual) MB_TRY(check_row_stride(what, "residual", a->residual_stride, a->rows, a->n));
  if (a->sum) MB_TRY(check_row_stride(what, "sum", a->sum_stride, a->rows, a->n));
  MB_TRY(check_row_stride(what, "y", a->y_stride, a->rows, a->n));
  if (a->y == a->sum && a->y) return fail(MIMIR_B200_E_INVALID, "%s: sum and y are one tensor", what);
  if ((a->sum && ((a->sum == a->x && a->sum_stride != a->x_stride) || (a->sum == a->residual && a->sum_stride != a->residual_stride))) ||
      (a->y && ((a->y == a->x && (a->y_stride != a->x_stride || a->y_type != a->type)) ||
                (a->y == a->residual && (a->y_stride != a->residual_stride || a->y_type != a->type)))))
    return fail(MIMIR_B200_E_INVALID, "%s: in place with another stride or type", what);
  return MIMIR_B200_OK;
}

int check_linear(const char* what, const MimirLinear* a, bool gated) {
  if (!a) return fail(MIMIR_B200_E_INVALID, "%s: null argument", what);
  if (a->type == MIMIR_B200_T_F32 || a->type == MIMIR_B200_T_I8) return fail(MIMIR_B200_E_UNSUPPORTED, "%s: operands are F16, BF16 or E4M3, not type %d", what, a->type);
  if (a->type != MIMIR_B200_T_F16 && a->type != MIMIR_B200_T_BF16 && a->type != MIMIR_B200_T_E4M3)
    return fail(MIMIR_B200_E_INVALID, "%s: unknown operand type %d", what, a->type);
  if (!row_type(a->out_type)) return fail(MIMIR_B200_E_INVALID, "%s: out is F32, F16 or BF16, not type %d", what, a->out_type);
  if (a->rows < 0 || a->n_in <= 0 || a->n_out <= 0) return fail(MIMIR_B200_E_INVALID, "%s: %d rows, %d in, %d out", what, a->rows, a->n_in, a->n_out);
  if (static_cast<long long>(a->rows) * a->n_out > (1LL << 40) || a->n_in > (1 << 24) || a->n_out > (1 << 24) || a->rows > (1 << 24))
    return fail(MIMIR_B200_E_INVALID, "%s: too many rows, inputs or features for one call", what);
  if (a->activation != -1 && (a->activation < MIMIR_B200_ELT_GELU || a->activation > MIMIR_B200_ELT_SIGMOID))
    return fail(MIMIR_B200_E_UNSUPPORTED, "%s: activation %d is none of a product's", what, a->activation);
  const bool coded = a->type == MIMIR_B200_T_E4M3;
  if (coded != (a->x_scale != nullptr) || coded != (a->w_scale != nullptr) || (coded && gated) != (a->up_scale != nullptr))
    return fail(MIMIR_B200_E_INVALID, "%s: scales belong to operands of type E4M3, each its own", what);
  if (!gated && (a->up || a->up_bias)) return fail(MIMIR_B200_E_INVALID, "%s: up belongs to gated_linear", what);
  if (gated && a->residual) return fail(MIMIR_B200_E_INVALID, "%s: a residual belongs to linear", what);
  const long long unit = 16 / type_bytes(a->type);
  MB_TRY(check_row_stride(what, "x", a->x_stride, a->rows, a->n_in));
  MB_TRY(check_row_stride(what, "w", a->w_stride, a->n_out, a->n_in));
  if (gated) MB_TRY(check_row_stride(what, "up", a->up_stride, a->n_out, a->n_in));
  if (a->residual) MB_TRY(check_row_stride(what, "residual", a->residual_stride, a->rows, a->n_out));
  MB_TRY(check_row_stride(what, "out", a->out_stride, a->rows, a->n_out));
  if (a->x_stride % unit || a->w_stride % unit || (gated && a->up_stride % unit))
    return fail(MIMIR_B200_E_UNSUPPORTED, "%s: strides of operands are multiples of 16 bytes", what);
  if (a->out && (a->out == a->x || a->out == a->w || a->out == a->up)) return fail(MIMIR_B200_E_INVALID, "%s: out is an operand", what);
  if (a->residual && a->residual == a->out && a->residual_stride != a->out_stride) return fail(MIMIR_B200_E_INVALID, "%s: in place with two strides", what);
  return MIMIR_B200_OK;
}

int run_linear(const char* what, const MimirLinear* a, bool gated, void* stream) {
  MB_TRY(check_linear(what, a, gated));
  MB_REQUIRE_INIT();
  if (a->rows == 0) return MIMIR_B200_OK;
  MB_TRY(check_device_pointer(what, "x", a->x));
  MB_TRY(check_device_pointer(what, "w", a->w));
  if (gated) MB_TRY(check_device_pointer(what, "up", a->up));
  if (!aligned16(a->x) || !aligned16(a->w) || (gated && !aligned16(a->up))) return fail(MIMIR_B200_E_UNSUPPORTED, "%s: operands start on 16 bytes", what);
  if (a->x_scale) MB_TRY(check_device_words(what, "x_scale", a->x_scale));
  if (a->w_scale) MB_TRY(check_device_words(what, "w_scale", a->w_scale));
  if (a->up_scale) MB_TRY(check_device_words(what, "up_scale", a->up_scale));
  if (a->bias) MB_TRY(check_device_words(what, "bias", a->bias));
  if (a->up_bias) MB_TRY(check_device_words(what, "up_bias", a->up_bias));
  if (a->residual) MB_TRY(check_device_pointer(what, "residual", a->residual));
  MB_TRY(check_device_pointer(what, "out", a->out));
  const int size = type_bytes(a->out_type);
  if (!on_boundary(a->out, size) || !on_boundary(a->residual, size)) return fail(MIMIR_B200_E_INVALID, "%s: misaligned pointer", what);
  return launch_linear(*a, gated, static_cast<cudaStream_t>(stream));
}

}  // namespace
}  // namespace mb

using namespace mb;

extern "C" {

int mimir_b200_dev_rope(const MimirRopePlan* plan, const int32_t* positions, const void* x, void* y, long long rows, int heads, int head_dim,
                        long long x_row_stride, long long x_head_stride, long long y_row_stride, long long y_head_stride, int type, void* stream) {
  if (!plan) return fail(MIMIR_B200_E_INVALID, "rope: null argument");
  if (plan->rot_dim <= 0 || (plan->rot_dim & 1) || plan->rot_dim > 2 * MIMIR_B200_MAX_ROPE_PAIRS)
    return fail(MIMIR_B200_E_INVALID, "rope: the plan was not made by rope_plan");
  if (rows < 0 || heads < 0 || head_dim <= 0 || plan->rot_dim > head_dim)
    return fail(MIMIR_B200_E_INVALID, "rope: %lld rows, %d heads of %d with %d turned", rows, heads, head_dim, plan->rot_dim);
  if (!row_type(type)) return fail(MIMIR_B200_E_INVALID, "rope: x and y are F32, F16 or BF16, not type %d", type);
  if (rows > 0x7fffffffLL || static_cast<long long>(heads) * head_dim > (1LL << 26)) return fail(MIMIR_B200_E_INVALID, "rope: too many rows or heads for one call");
  if (x_row_stride < 0 || x_head_stride < 0 || y_row_stride < 0 || y_head_stride < 0) return fail(MIMIR_B200_E_INVALID, "rope: negative stride");
  if (x == y && (x_row_stride != y_row_stride || x_head_stride != y_head_stride)) return fail(MIMIR_B200_E_INVALID, "rope: in place with two sets of strides");
  MB_REQUIRE_INIT();
  if (rows == 0 || heads == 0) return MIMIR_B200_OK;
  MB_TRY(check_device_words("rope", "positions", positions));
  MB_TRY(check_device_pointer("rope", "x", x));
  MB_TRY(check_device_pointer("rope", "y", y));
  const uintptr_t size = static_cast<uintptr_t>(type_bytes(type));
  if (reinterpret_cast<uintptr_t>(x) % size || reinterpret_cast<uintptr_t>(y) % size) return fail(MIMIR_B200_E_INVALID, "rope: misaligned pointer");
  RopeLaunch r = {};
  r.plan = *plan, r.positions = positions, r.x = x, r.y = y, r.rows = rows, r.heads = heads, r.dim = head_dim, r.type = type;
  r.x_row = x_row_stride, r.x_head = x_head_stride, r.y_row = y_row_stride, r.y_head = y_head_stride;
  return launch_rope(r, static_cast<cudaStream_t>(stream));
}

int mimir_b200_dev_cache_write(const MimirPagedCache* cache, const MimirPagedBatch* batch, const void* k, const void* v, int type,
                               long long row_stride, long long head_stride, void* stream) {
  MB_TRY(check_sizes("cache_write", cache, batch));
  if (!row_type(type)) return fail(MIMIR_B200_E_INVALID, "cache_write: rows are F32, F16 or BF16, not type %d", type);
  MB_REQUIRE_INIT();
  if (batch->n_seqs == 0 || batch->n_rows == 0) return MIMIR_B200_OK;
  PagedView p = {};
  MB_TRY(check_row_tensors("cache_write", k, v, type, row_stride, head_stride));
  MB_TRY(check_pointers("cache_write", cache, batch, &p, true));
  return launch_cache_write(p, cache->type, k, v, type, row_stride, head_stride, static_cast<cudaStream_t>(stream));
}

int mimir_b200_dev_cache_read(const MimirPagedCache* cache, const MimirPagedBatch* batch, const int32_t* out_start, int out_rows, void* k, void* v,
                              int type, long long row_stride, long long head_stride, void* stream) {
  MB_TRY(check_sizes("cache_read", cache, batch));
  if (!row_type(type)) return fail(MIMIR_B200_E_INVALID, "cache_read: rows are F32, F16 or BF16, not type %d", type);
  if (out_rows < 0) return fail(MIMIR_B200_E_INVALID, "cache_read: negative out_rows");
  MB_REQUIRE_INIT();
  if (batch->n_seqs == 0 || out_rows == 0) return MIMIR_B200_OK;
  PagedView p = {};
  MB_TRY(check_row_tensors("cache_read", k, v, type, row_stride, head_stride));
  MB_TRY(check_pointers("cache_read", cache, batch, &p, false));
  MB_TRY(check_device_words("cache_read", "out_start", out_start));
  return launch_cache_read(p, cache->type, out_start, out_rows, k, v, type, row_stride, head_stride, static_cast<cudaStream_t>(stream));
}

int mimir_b200_paged_attention_workspace(const MimirPagedCache* cache, const MimirPagedBatch* batch, const MimirPagedAttention* attention,
                                         uint64_t* bytes) {
  if (!bytes) return fail(MIMIR_B200_E_INVALID, "paged_attention_workspace: null argument");
  AttendLaunch l = {};
  MB_TRY(check_attention("paged_attention_workspace", cache, batch, attention, &l));
  MB_REQUIRE_INIT();
  *bytes = (l.p.n_seqs == 0 || l.p.n_rows == 0 || l.p.max_rows == 0) ? 0 : paged_attention_ws_bytes(l);
  return MIMIR_B200_OK;
}

int mimir_b200_dev_paged_attention(const MimirPagedCache* cache, const MimirPagedBatch* batch, const MimirPagedAttention* attention, void* stream) {
  AttendLaunch l = {};
  MB_TRY(check_attention("paged_attention", cache, batch, attention, &l));
  MB_REQUIRE_INIT();
  if (l.p.n_seqs == 0 || l.p.n_rows == 0 || l.p.max_rows == 0) return MIMIR_B200_OK;
  const int max_rows = l.p.max_rows, max_kv = l.p.max_kv;
  MB_TRY(check_device_pointer("paged_attention", "q", l.q));
  MB_TRY(check_device_pointer("paged_attention", "out", l.out));
  if (l.lse) MB_TRY(check_device_words("paged_attention", "lse", l.lse));
  if (l.ws) MB_TRY(check_device_pointer("paged_attention", "workspace", l.ws));
  if (!aligned16(l.q) || !aligned16(l.out) || !aligned16(l.ws))
    return fail(MIMIR_B200_E_UNSUPPORTED, "paged_attention: q, out and workspace start on 16 bytes");
  MB_TRY(check_pointers("paged_attention", cache, batch, &l.p, true));
  l.p.max_rows = max_rows, l.p.max_kv = max_kv;
  return launch_paged_attention(l, static_cast<cudaStream_t>(stream));
}

int mimir_b200_dev_sample_rows(const void* logits, int type, long long rows, int n, long long row_stride, const float* temperature,
                               const int32_t* top_k, const float* top_p, const float* min_p, const float* uniform, int32_t* ids, float* logprob,
                               void* stream) {
  if (!row_type(type)) return fail(MIMIR_B200_E_INVALID, "sample_rows: logits are F32, F16 or BF16, not type %d", type);
  if (rows < 0 || n <= 0 || n > (1 << 24) || rows > 0x7fffffffLL) return fail(MIMIR_B200_E_INVALID, "sample_rows: %lld rows of %d logits", rows, n);
  if (row_stride < 0) return fail(MIMIR_B200_E_INVALID, "sample_rows: negative stride");
  MB_REQUIRE_INIT();
  if (rows == 0) return MIMIR_B200_OK;
  MB_TRY(check_device_pointer("sample_rows", "logits", logits));
  MB_TRY(check_device_words("sample_rows", "uniform", uniform));
  MB_TRY(check_device_words("sample_rows", "ids", ids));
  if (temperature) MB_TRY(check_device_words("sample_rows", "temperature", temperature));
  if (top_k) MB_TRY(check_device_words("sample_rows", "top_k", top_k));
  if (top_p) MB_TRY(check_device_words("sample_rows", "top_p", top_p));
  if (min_p) MB_TRY(check_device_words("sample_rows", "min_p", min_p));
  if (logprob) MB_TRY(check_device_words("sample_rows", "logprob", logprob));
  if (reinterpret_cast<uintptr_t>(logits) % static_cast<uintptr_t>(type_bytes(type))) return fail(MIMIR_B200_E_INVALID, "sample_rows: misaligned logits");
  SampleLaunch s = {};
  s.x = logits, s.rows = rows, s.row_stride = row_stride, s.n = n, s.type = type;
  s.temperature = temperature, s.top_k = top_k, s.top_p = top_p, s.min_p = min_p, s.uniform = uniform, s.ids = ids, s.logprob = logprob;
  return launch_sample_rows(s, static_cast<cudaStream_t>(stream));
}

int mimir_b200_dev_norm_rows(const MimirNormRows* norm, void* stream) {
  MB_TRY(check_norm_rows(norm));
  MB_REQUIRE_INIT();
  if (norm->rows == 0) return MIMIR_B200_OK;
  MB_TRY(check_device_pointer("norm_rows", "x", norm->x));
  MB_TRY(check_device_pointer("norm_rows", "y", norm->y));
  if (norm->residual) MB_TRY(check_device_pointer("norm_rows", "residual", norm->residual));
  if (norm->sum) MB_TRY(check_device_pointer("norm_rows", "sum", norm->sum));
  if (norm->gamma) MB_TRY(check_device_words("norm_rows", "gamma", norm->gamma));
  if (norm->y_scale) MB_TRY(check_device_words("norm_rows", "y_scale", norm->y_scale));
  const int size = type_bytes(norm->type);
  if (!on_boundary(norm->x, size) || !on_boundary(norm->residual, size) || !on_boundary(norm->sum, size) || !on_boundary(norm->y, type_bytes(norm->y_type)))
    return fail(MIMIR_B200_E_INVALID, "norm_rows: misaligned pointer");
  return launch_norm_rows(*norm, static_cast<cudaStream_t>(stream));
}

int mimir_b200_dev_linear(const MimirLinear* linear, void* stream) { return run_linear("linear", linear, false, stream); }
int mimir_b200_dev_gated_linear(const MimirLinear* linear, void* stream) { return run_linear("gated_linear", linear, true, stream); }

}  // extern "C"
