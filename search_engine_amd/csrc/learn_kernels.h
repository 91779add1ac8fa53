// Launchers of the kernels that learn from clicks: the pooled row lookup with its gradients
// (learn_lookup.hip) and the cross entropy of queries over a corpus with its gradients
// (learn_xent.hip). Arguments have been checked by learn_runtime.hip. Nothing here allocates,
// waits or keeps anything between calls: everything goes to the caller's buffers and stream.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace vs {
namespace learn {

// A table of rows in device memory. Strides are in elements.
struct Table {
    const void* rows;
    uint64_t stride;
    uint64_t n_rows;
    uint32_t dim;
    int32_t dtype;      // VS_F32 or VS_BF16
    const uint64_t* present;  // rows that exist, bit r & 63 of word r >> 6; null = all
    uint32_t first_id;  // the id of row 0
};

// The ids of a pooled lookup: bag b holds positions [offsets[b], offsets[b + 1]) (offsets null: position b alone).
struct Bags {
    const uint32_t* ids;
    uint64_t n_ids;
    const uint32_t* offsets;
    uint64_t n_bags;
    const float* weights;  // null = 1
    float scale;
};

hipError_t launch_lookup(const Table& t, const Bags& b, void* out, int32_t out_dtype, uint64_t out_stride,
                         hipStream_t stream);

uint64_t lookup_grad_workspace_bytes(uint64_t n_ids, uint64_t n_rows, uint32_t dim);
struct RowGrads {
    void* rows;
    int32_t dtype;
    uint64_t stride;
    uint32_t* unique;  // null: row r is added to rows[r]; else the k-th smallest id's sum is rows[k]
    uint32_t* count;
};
hipError_t launch_lookup_grad(const void* grad_out, int32_t dtype, uint64_t grad_stride, uint32_t dim, const Bags& b,
                              uint64_t n_rows, void* workspace, const RowGrads& out, hipStream_t stream);
hipError_t launch_lookup_grad_weights(const Table& t, const Bags& b, const void* grad_out, int32_t grad_dtype,
                                      uint64_t grad_stride, float* out, hipStream_t stream);

// The cross entropy of n_q queries over the candidates of a table.
struct Xent {
    Table t;
    const void* queries;  // of the table's type, or f32 (queries_f32): rounded to it
    bool queries_f32;
    uint64_t query_stride;
    uint32_t n_q;
    const uint32_t* targets;  // ids
    const uint64_t* mask;     // candidates, null = all
    const float* norms;       // not null: the rows' lengths; logits are scale * cosine
    float scale;
};
// What a call needs: the loss, or the gradients, of n_q queries over rows of this layout (`aligned`: read straight from the
// table, see rows_are_aligned).
uint64_t xent_workspace_bytes(uint32_t n_q, uint64_t n_rows, uint32_t dim, int32_t dtype, bool aligned, bool gradients);
// Whether rows are whole 16-byte chunks at multiples of 16 bytes; others are copied to such, in the workspace.
bool rows_are_aligned(const Table& t);
hipError_t launch_xent(const Xent& x, void* workspace, float* loss, float* lse, hipStream_t stream);
// (gradients are of the queries' and the rows' types)
hipError_t launch_xent_grad(const Xent& x, const float* loss, const float* lse, const float* grad_loss, void* workspace,
                            void* grad_queries, uint64_t grad_query_stride, void* grad_rows, uint64_t grad_row_stride,
                            hipStream_t stream);

}  // namespace learn
}  // namespace vs
