// The entry points that learn from clicks (declared in include/vs_abi.h): argument checks, the snapshot of a store,
// and the launches of learn_lookup.hip and learn_xent.hip. No computation happens here.
#include <algorithm>

#include "learn_kernels.h"
#include "vs_internal.h"

using vsrt::fail;
using vsrt::Snapshot;
namespace learn = vs::learn;

namespace {

bool is_float(int32_t dtype) { return dtype == VS_F32 || dtype == VS_BF16; }
uint64_t size_of(int32_t dtype) { return dtype == VS_F32 ? 4 : 2; }

// A matrix of the caller's: `what` names it in the error.
int32_t check_matrix(const char* what, const void* p, int32_t dtype, uint64_t n_rows, uint64_t stride, uint32_t dim) {
    if (!is_float(dtype)) return fail(VS_E_INVALID_ARG, "%s: element type %d is not VS_F32 or VS_BF16", what, dtype);
    if (dim == 0 || dim > VS_LEARN_MAX_DIM) return fail(VS_E_INVALID_ARG, "%s: dimension %u out of range", what, dim);
    if (!p && n_rows) return fail(VS_E_INVALID_ARG, "%s: null device buffer", what);
    if ((uintptr_t)p % size_of(dtype)) return fail(VS_E_INVALID_ARG, "%s: address is not aligned to its elements", what);
    if (stride < dim) return fail(VS_E_INVALID_ARG, "%s: stride %llu is less than the dimension %u", what, (unsigned long long)stride, dim);
    if (n_rows && stride > (1ull << 60) / n_rows)
        return fail(VS_E_INVALID_ARG, "%s: %llu rows of stride %llu are no device memory", what, (unsigned long long)n_rows, (unsigned long long)stride);
    return VS_OK;
}

// Last of all checks, and makes the context's GPU current.
int32_t use_ctx(vs_ctx* ctx) {
    if (!ctx) return fail(VS_E_INVALID_ARG, "null context");
    HIP_TRY(hipSetDevice(ctx->device));
    return VS_OK;
}

int32_t check_table(const void* rows, int32_t dtype, uint64_t n_rows, uint64_t stride, uint32_t dim) {
    if (n_rows == 0 || n_rows > VS_LEARN_MAX_ROWS) return fail(VS_E_INVALID_ARG, "rows: a table of %llu rows", (unsigned long long)n_rows);
    return check_matrix("rows", rows, dtype, n_rows, stride, dim);
}

int32_t check_bags(const uint32_t* ids, uint64_t n_ids, uint64_t n_bags) {
    if (n_ids > VS_LOOKUP_MAX_IDS) return fail(VS_E_INVALID_ARG, "%llu ids are more than %u", (unsigned long long)n_ids, VS_LOOKUP_MAX_IDS);
    if (n_bags > VS_LOOKUP_MAX_IDS) return fail(VS_E_INVALID_ARG, "%llu bags are more than %u", (unsigned long long)n_bags, VS_LOOKUP_MAX_IDS);
    if (!ids && n_ids) return fail(VS_E_INVALID_ARG, "ids: null device buffer");
    return VS_OK;
}

int32_t check_workspace(const void* p, uint64_t have, uint64_t need, const char* ask) {
    if (have < need)
        return fail(VS_E_CAPACITY, "workspace of %llu bytes, the call needs %llu (%s)", (unsigned long long)have, (unsigned long long)need, ask);
    if (!p && need) return fail(VS_E_INVALID_ARG, "workspace: null device buffer");
    return VS_OK;
}

int32_t check_queries(uint32_t n_q) {
    if (n_q > VS_XENT_MAX_QUERIES) return fail(VS_E_INVALID_ARG, "n_q = %u out of range", n_q);
    return VS_OK;
}

int32_t make_table(const void* rows, int32_t dtype, uint64_t n_rows, uint64_t stride, uint32_t dim, learn::Table* t) {
    if (int32_t rc = check_table(rows, dtype, n_rows, stride, dim)) return rc;
    *t = learn::Table{rows, stride, n_rows, dim, dtype, nullptr, 0};
    return VS_OK;
}

// The sealed rows of a store, as registered in a snapshot.
learn::Table table_of(const vs::SlabView& v) {
    const uint64_t padded = (uint64_t)v.row_vecs * 16 / size_of(v.dtype);  // columns from `dim` on are zero
    return learn::Table{v.rows, padded, v.n_slots, v.dim, v.dtype, v.present, v.docid_base};
}

int32_t check_sealed(vs_store* s) {
    if (int32_t rc = vsrt::check_store(s)) return rc;
    if (!s->sealed.load()) return fail(VS_E_NOT_SEALED, "store %u was never sealed", s->index);
    if (!is_float(s->dtype)) return fail(VS_E_INVALID_ARG, "store %u holds no f32 or bf16 rows", s->index);
    if (s->capacity > VS_LEARN_MAX_ROWS) return fail(VS_E_INVALID_ARG, "store %u has more than %u slots", s->index, VS_LEARN_MAX_ROWS);
    return VS_OK;
}

int32_t check_store_xent(vs_store* s, const void* queries, uint32_t n_q, uint32_t dim, const void* targets) {
    if (int32_t rc = check_sealed(s)) return rc;
    if (int32_t rc = vsrt::check_device_search(s, dim, 1)) return rc;
    if (s->metric != VS_ANGULAR && s->metric != VS_DOT)
        return fail(VS_E_INVALID_ARG, "store %u: the loss is defined for VS_ANGULAR and VS_DOT", s->index);
    if (int32_t rc = check_queries(n_q)) return rc;
    if (n_q && (!queries || !targets)) return fail(VS_E_INVALID_ARG, "null device buffer");
    return VS_OK;
}

learn::Xent xent_of(const vs::SlabView& v, const float* queries, uint32_t n_q, const uint32_t* targets, const uint64_t* mask, float scale) {
    learn::Xent x{};
    x.t = table_of(v);
    x.queries = queries;
    x.queries_f32 = true;
    x.query_stride = v.dim;
    x.n_q = n_q;
    x.targets = targets;
    x.mask = mask;
    x.norms = v.metric == VS_ANGULAR ? v.norms : nullptr;
    x.scale = scale;
    return x;
}

// Runs `body` (which returns a hipError_t) over the registered rows of a sealed store on the caller's stream.
template <typename F>
int32_t over_store(vs_store* s, hipStream_t stream, F&& body) {
    // (the event that a later seal waits for would become part of the graph, and the store's buffers of today with it)
    hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
    HIP_TRY(hipStreamIsCapturing(stream, &capture));
    if (capture != hipStreamCaptureStatusNone)
        return fail(VS_E_INVALID_ARG, "store %u: the call may not be recorded into a graph", s->index);
    Snapshot snap;
    vsrt::snapshot_begin(s, &snap);
    const int32_t rc = body(snap.v);
    const int32_t rc2 = vsrt::snapshot_end_async(s, &snap, stream, true);
    return rc ? rc : rc2;
}

int32_t status(hipError_t e, const char* what) {
    return e == hipSuccess ? VS_OK : fail(VS_E_DEVICE, "%s failed: %s", what, hipGetErrorString(e));
}

hipStream_t stream_of(void* s) { return static_cast<hipStream_t>(s); }

// Enough for the loss and the gradients both.
uint64_t xent_bytes(uint32_t n_q, uint64_t n_rows, uint32_t dim, int32_t dtype, bool aligned) {
    if (!n_q) return 0;
    return std::max(learn::xent_workspace_bytes(n_q, n_rows, dim, dtype, aligned, false),
                    learn::xent_workspace_bytes(n_q, n_rows, dim, dtype, aligned, true));
}
uint64_t xent_bytes(const learn::Table& t, uint32_t n_q, bool gradients) {
    return n_q ? learn::xent_workspace_bytes(n_q, t.n_rows, t.dim, t.dtype, learn::rows_are_aligned(t), gradients) : 0;
}

// vs_xent_device and vs_xent_grad_device share their arguments.
int32_t make_xent(const void* queries, uint32_t n_q, uint64_t query_stride, const void* rows, uint64_t n_rows,
                  uint64_t row_stride, int32_t dtype, uint32_t dim, const uint32_t* targets, const uint64_t* mask, float scale,
                  const void* workspace, uint64_t workspace_bytes, bool gradients, learn::Xent* x) {
    *x = learn::Xent{};
    if (int32_t rc = make_table(rows, dtype, n_rows, row_stride, dim, &x->t)) return rc;
    if (int32_t rc = check_queries(n_q)) return rc;
    if (int32_t rc = check_matrix("queries", queries, dtype, n_q, query_stride, dim)) return rc;
    if (n_q && !targets) return fail(VS_E_INVALID_ARG, "targets: null device buffer");
    if (int32_t rc = check_workspace(workspace, workspace_bytes, xent_bytes(x->t, n_q, gradients), "vs_xent_workspace_bytes"))
        return rc;
    x->queries = queries;
    x->queries_f32 = dtype == VS_F32;
    x->query_stride = query_stride;
    x->n_q = n_q;
    x->targets = targets;
    x->mask = mask;
    x->scale = scale;
    return VS_OK;
}

}  // namespace

// ---- lookup -----------------------------------------------------------------------

extern "C" int32_t vs_lookup_device(vs_ctx* ctx, const void* d_rows, int32_t dtype, uint64_t n_rows, uint64_t row_stride,
                                    uint32_t dim, const uint32_t* d_ids, uint64_t n_ids, const uint32_t* d_offsets,
                                    uint64_t n_bags, const float* d_weights, float scale, void* d_out, int32_t out_dtype,
                                    uint64_t out_stride, void* hip_stream) {
    learn::Table t;
    if (int32_t rc = make_table(d_rows, dtype, n_rows, row_stride, dim, &t)) return rc;
    if (int32_t rc = check_bags(d_ids, n_ids, n_bags)) return rc;
    if (int32_t rc = check_matrix("out", d_out, out_dtype, n_bags, out_stride, dim)) return rc;
    if (int32_t rc = use_ctx(ctx)) return rc;
    return status(learn::launch_lookup(t, {d_ids, n_ids, d_offsets, n_bags, d_weights, scale}, d_out, out_dtype, out_stride,
                                       stream_of(hip_stream)), "lookup");
}

extern "C" int32_t vs_store_lookup_device(vs_store* s, const uint32_t* d_ids, uint64_t n_ids, const uint32_t* d_offsets,
                                          uint64_t n_bags, const float* d_weights, float scale, void* d_out,
                                          int32_t out_dtype, uint64_t out_stride, void* hip_stream) {
    if (int32_t rc = check_sealed(s)) return rc;
    if (int32_t rc = check_bags(d_ids, n_ids, n_bags)) return rc;
    if (int32_t rc = check_matrix("out", d_out, out_dtype, n_bags, out_stride, s->dim)) return rc;
    hipStream_t stream = stream_of(hip_stream);
    return over_store(s, stream, [&](const vs::SlabView& v) {
        return status(learn::launch_lookup(table_of(v), {d_ids, n_ids, d_offsets, n_bags, d_weights, scale}, d_out, out_dtype,
                                           out_stride, stream), "lookup");
    });
}

extern "C" int32_t vs_lookup_grad_workspace_bytes(vs_ctx* ctx, uint64_t n_ids, uint64_t n_rows, uint32_t dim, uint64_t* bytes) {
    if (!bytes) return fail(VS_E_INVALID_ARG, "null argument");
    if (n_ids > VS_LOOKUP_MAX_IDS) return fail(VS_E_INVALID_ARG, "%llu ids are more than %u", (unsigned long long)n_ids, VS_LOOKUP_MAX_IDS);
    if (n_rows == 0 || n_rows > VS_LEARN_MAX_ROWS) return fail(VS_E_INVALID_ARG, "rows: a table of %llu rows", (unsigned long long)n_rows);
    if (dim == 0 || dim > VS_LEARN_MAX_DIM) return fail(VS_E_INVALID_ARG, "dimension %u out of range", dim);
    if (!ctx) return fail(VS_E_INVALID_ARG, "null context");
    *bytes = learn::lookup_grad_workspace_bytes(n_ids, n_rows, dim);
    return VS_OK;
}

extern "C" int32_t vs_lookup_grad_device(vs_ctx* ctx, const void* d_grad_out, int32_t dtype, uint64_t grad_out_stride,
                                         uint32_t dim, const uint32_t* d_ids, uint64_t n_ids, const uint32_t* d_offsets,
                                         uint64_t n_bags, const float* d_weights, float scale, uint64_t n_rows,
                                         void* d_workspace, uint64_t workspace_bytes, void* d_grad_rows,
                                         int32_t grad_rows_dtype, uint64_t grad_rows_stride, uint32_t* d_unique_ids,
                                         uint32_t* d_n_unique, void* hip_stream) {
    if (int32_t rc = check_bags(d_ids, n_ids, n_bags)) return rc;
    if (int32_t rc = check_matrix("grad_out", d_grad_out, dtype, n_bags, grad_out_stride, dim)) return rc;
    if (!d_unique_ids != !d_n_unique) return fail(VS_E_INVALID_ARG, "unique_ids and n_unique: one without the other");
    if (n_rows == 0 || n_rows > VS_LEARN_MAX_ROWS) return fail(VS_E_INVALID_ARG, "rows: a table of %llu rows", (unsigned long long)n_rows);
    if (int32_t rc = check_matrix("grad_rows", d_grad_rows, grad_rows_dtype, d_unique_ids ? n_ids : n_rows, grad_rows_stride, dim)) return rc;
    if (int32_t rc = check_workspace(d_workspace, workspace_bytes, learn::lookup_grad_workspace_bytes(n_ids, n_rows, dim),
                                     "vs_lookup_grad_workspace_bytes"))
        return rc;
    if (int32_t rc = use_ctx(ctx)) return rc;
    return status(learn::launch_lookup_grad(d_grad_out, dtype, grad_out_stride, dim, {d_ids, n_ids, d_offsets, n_bags, d_weights, scale},
                                            n_rows, d_workspace, {d_grad_rows, grad_rows_dtype, grad_rows_stride, d_unique_ids, d_n_unique},
                                            stream_of(hip_stream)), "lookup gradient");
}

extern "C" int32_t vs_lookup_grad_weights_device(vs_ctx* ctx, const void* d_rows, int32_t dtype, uint64_t n_rows,
                                                 uint64_t row_stride, uint32_t dim, const uint32_t* d_ids, uint64_t n_ids,
                                                 const uint32_t* d_offsets, uint64_t n_bags, float scale,
                                                 const void* d_grad_out, int32_t grad_dtype, uint64_t grad_out_stride,
                                                 float* d_grad_weights, void* hip_stream) {
    learn::Table t;
    if (int32_t rc = make_table(d_rows, dtype, n_rows, row_stride, dim, &t)) return rc;
    if (int32_t rc = check_bags(d_ids, n_ids, n_bags)) return rc;
    if (int32_t rc = check_matrix("grad_out", d_grad_out, grad_dtype, n_bags, grad_out_stride, dim)) return rc;
    if (!d_grad_weights && n_ids) return fail(VS_E_INVALID_ARG, "grad_weights: null device buffer");
    if (int32_t rc = use_ctx(ctx)) return rc;
    return status(learn::launch_lookup_grad_weights(t, {d_ids, n_ids, d_offsets, n_bags, nullptr, scale}, d_grad_out, grad_dtype,
                                                    grad_out_stride, d_grad_weights, stream_of(hip_stream)), "lookup gradient");
}

// ---- cross entropy ------------------------------------------------------------------

extern "C" int32_t vs_xent_workspace_bytes(vs_ctx* ctx, uint32_t n_q, uint64_t n_rows, uint32_t dim, int32_t dtype, uint64_t* bytes) {
    if (!bytes) return fail(VS_E_INVALID_ARG, "null argument");
    if (int32_t rc = check_queries(n_q)) return rc;
    if (n_rows == 0 || n_rows > VS_LEARN_MAX_ROWS) return fail(VS_E_INVALID_ARG, "rows: a table of %llu rows", (unsigned long long)n_rows);
    if (dim == 0 || dim > VS_LEARN_MAX_DIM) return fail(VS_E_INVALID_ARG, "dimension %u out of range", dim);
    if (!is_float(dtype)) return fail(VS_E_INVALID_ARG, "element type %d is not VS_F32 or VS_BF16", dtype);
    if (!ctx) return fail(VS_E_INVALID_ARG, "null context");
    *bytes = xent_bytes(n_q, n_rows, dim, dtype, false);
    return VS_OK;
}

extern "C" int32_t vs_xent_call_workspace_bytes(vs_ctx* ctx, uint32_t n_q, const void* d_rows, uint64_t n_rows, uint64_t row_stride,
                                                int32_t dtype, uint32_t dim, int32_t gradients, uint64_t* bytes) {
    if (!bytes) return fail(VS_E_INVALID_ARG, "null argument");
    learn::Table t;
    if (int32_t rc = check_queries(n_q)) return rc;
    if (int32_t rc = make_table(d_rows, dtype, n_rows, row_stride, dim, &t)) return rc;
    if (!ctx) return fail(VS_E_INVALID_ARG, "null context");
    *bytes = xent_bytes(t, n_q, gradients != 0);
    return VS_OK;
}

extern "C" int32_t vs_xent_device(vs_ctx* ctx, const void* d_queries, uint32_t n_q, uint64_t query_stride, const void* d_rows,
                                  uint64_t n_rows, uint64_t row_stride, int32_t dtype, uint32_t dim, const uint32_t* d_targets,
                                  const uint64_t* d_mask_words, float scale, void* d_workspace, uint64_t workspace_bytes,
                                  float* d_loss, float* d_lse, void* hip_stream) {
    learn::Xent x;
    if (int32_t rc = make_xent(d_queries, n_q, query_stride, d_rows, n_rows, row_stride, dtype, dim, d_targets, d_mask_words,
                               scale, d_workspace, workspace_bytes, false, &x))
        return rc;
    if (n_q && (!d_loss || !d_lse)) return fail(VS_E_INVALID_ARG, "loss or lse: null device buffer");
    if (int32_t rc = use_ctx(ctx)) return rc;
    if (!n_q) return VS_OK;
    return status(learn::launch_xent(x, d_workspace, d_loss, d_lse, stream_of(hip_stream)), "cross entropy");
}

extern "C" int32_t vs_xent_grad_device(vs_ctx* ctx, const void* d_queries, uint32_t n_q, uint64_t query_stride, const void* d_rows,
                                       uint64_t n_rows, uint64_t row_stride, int32_t dtype, uint32_t dim, const uint32_t* d_targets,
                                       const uint64_t* d_mask_words, float scale, const float* d_loss, const float* d_lse,
                                       const float* d_grad_loss, void* d_workspace, uint64_t workspace_bytes, void* d_grad_queries,
                                       void* d_grad_rows, void* hip_stream) {
    learn::Xent x;
    if (int32_t rc = make_xent(d_queries, n_q, query_stride, d_rows, n_rows, row_stride, dtype, dim, d_targets, d_mask_words,
                               scale, d_workspace, workspace_bytes, true, &x))
        return rc;
    if (n_q && (!d_loss || !d_lse)) return fail(VS_E_INVALID_ARG, "loss or lse: null device buffer");
    for (const void* p : {(const void*)d_grad_queries, (const void*)d_grad_rows})
        if ((uintptr_t)p % size_of(dtype)) return fail(VS_E_INVALID_ARG, "gradients: address is not aligned to its elements");
    if (int32_t rc = use_ctx(ctx)) return rc;
    return status(learn::launch_xent_grad(x, d_loss, d_lse, d_grad_loss, d_workspace, d_grad_queries, query_stride,
                                          d_grad_rows, row_stride, stream_of(hip_stream)), "cross entropy gradient");
}

extern "C" int32_t vs_store_xent_workspace_bytes(vs_store* s, uint32_t n_q, uint64_t* bytes) {
    if (!s || !bytes) return fail(VS_E_INVALID_ARG, "null argument");
    if (!is_float(s->dtype)) return fail(VS_E_INVALID_ARG, "store %u holds no f32 or bf16 rows", s->index);
    if (int32_t rc = check_queries(n_q)) return rc;
    const learn::Table t = table_of(s->view(0));
    *bytes = std::max(xent_bytes(t, n_q, false), xent_bytes(t, n_q, true));
    return VS_OK;
}

extern "C" int32_t vs_store_xent_call_workspace_bytes(vs_store* s, uint32_t n_q, int32_t gradients, uint64_t* bytes) {
    if (!s || !bytes) return fail(VS_E_INVALID_ARG, "null argument");
    if (!is_float(s->dtype)) return fail(VS_E_INVALID_ARG, "store %u holds no f32 or bf16 rows", s->index);
    if (int32_t rc = check_queries(n_q)) return rc;
    *bytes = xent_bytes(table_of(s->view(0)), n_q, gradients != 0);
    return VS_OK;
}

extern "C" int32_t vs_store_xent_device(vs_store* s, const float* d_queries, uint32_t n_q, uint32_t dim, const uint32_t* d_targets,
                                        const uint64_t* d_mask_words, float scale, void* d_workspace, uint64_t workspace_bytes,
                                        float* d_loss, float* d_lse, void* hip_stream) {
    if (int32_t rc = check_store_xent(s, d_queries, n_q, dim, d_targets)) return rc;
    if (!n_q) return VS_OK;
    if (!d_loss || !d_lse) return fail(VS_E_INVALID_ARG, "loss or lse: null device buffer");
    hipStream_t stream = stream_of(hip_stream);
    return over_store(s, stream, [&](const vs::SlabView& v) {
        if (int32_t rc = check_workspace(d_workspace, workspace_bytes, xent_bytes(table_of(v), n_q, false), "vs_store_xent_workspace_bytes"))
            return rc;
        return status(learn::launch_xent(xent_of(v, d_queries, n_q, d_targets, d_mask_words, scale), d_workspace, d_loss, d_lse, stream),
                      "cross entropy");
    });
}

extern "C" int32_t vs_store_xent_grad_device(vs_store* s, const float* d_queries, uint32_t n_q, uint32_t dim, const uint32_t* d_targets,
                                             const uint64_t* d_mask_words, float scale, const float* d_loss, const float* d_lse,
                                             const float* d_grad_loss, void* d_workspace, uint64_t workspace_bytes,
                                             float* d_grad_queries, void* hip_stream) {
    if (int32_t rc = check_store_xent(s, d_queries, n_q, dim, d_targets)) return rc;
    if (!n_q) return VS_OK;
    if (!d_loss || !d_lse || !d_grad_queries) return fail(VS_E_INVALID_ARG, "loss, lse or grad_queries: null device buffer");
    hipStream_t stream = stream_of(hip_stream);
    return over_store(s, stream, [&](const vs::SlabView& v) {
        if (int32_t rc = check_workspace(d_workspace, workspace_bytes, xent_bytes(table_of(v), n_q, true), "vs_store_xent_workspace_bytes"))
            return rc;
        return status(learn::launch_xent_grad(xent_of(v, d_queries, n_q, d_targets, d_mask_words, scale), d_loss, d_lse, d_grad_loss,
                                              d_workspace, d_grad_queries, v.dim, nullptr, 0, stream), "cross entropy gradient");
    });
}
