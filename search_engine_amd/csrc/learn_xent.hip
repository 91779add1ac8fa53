// The cross entropy of queries over a whole corpus, and its gradients, without keeping the logits.
//
//   z[q][j] = scale * <query q, row j> for every candidate row j (or scale * cosine, where norms are given)
//   others  = sum over j != t of exp(z[q][j]),  t = the clicked row
//   loss[q] = log(1 + others / exp(z[q][t])),   lse[q] = log(others + exp(z[q][t]))
//   G[q][j] = grad_loss[q] * scale * exp(z[q][j] - lse[q]),  G[q][t] = grad_loss[q] * scale * expm1(-loss[q])
//   dqueries = G rows,  drows = transpose(G) queries
//
// The clicked row is kept out of the sum so that a loss near zero, and the gradient p[t] - 1 with it, keep their
// digits: neither is a difference of nearly equal numbers. A query whose click is no candidate has loss 0 and gradients 0.
//
// Under a filter the candidates are listed first, and everything reads through the list: a row that is no candidate is
// never read (whatever it holds), and costs nothing.
#include "../../include/vs_abi.h"
#include "learn_kernels.h"
#include "learn_device.h"

namespace vs {
namespace learn {
namespace {

constexpr uint32_t NONE = 0xFFFFFFFFu;

struct XentArgs {
    Table t;
    const uint32_t* list;   // candidate rows, ascending; null = every row
    const uint32_t* count;  // of the list
    const float* norms;
    const void* q;          // [n_q][kp] of the table's type, zero from `dim` on
    uint32_t kp, n_q;
    const uint32_t* click;  // [n_q] place of the clicked row among the candidates, or NONE
    const float* qscale;    // [n_q] factor of a query's products
    // loss
    float* part_m;          // [splits][n_q]
    float* part_l;
    float* click_z;         // [n_q]
    // gradients
    const float* lse;
    const float* loss;
    const float* grad_loss;
    float* g;               // [piece][n_q]
    uint32_t piece_begin, piece_rows;
    void* grad_rows;
    uint64_t grad_row_stride;
    float* part_q;          // [splits][n_q][dim]
    uint32_t splits;
    bool first_piece;
};

__device__ __forceinline__ uint32_t candidates(const XentArgs& a) { return a.list ? *a.count : (uint32_t)a.t.n_rows; }
__device__ __forceinline__ uint64_t row_at(const XentArgs& a, uint32_t place) { return a.list ? a.list[place] : place; }

// ---- candidates and queries ------------------------------------------------------------------

__device__ __forceinline__ uint64_t word_at(const uint64_t* mask, const uint64_t* present, uint64_t i, uint64_t n_rows) {
    uint64_t w = mask ? mask[i] : ~0ull;
    if (present) w &= present[i];
    const uint64_t left = n_rows - i * 64;
    return left < 64 ? w & ((1ull << left) - 1) : w;
}

// The candidate rows in ascending order: 1024 words of the masks per workgroup, which counts the words before its own
// by itself (at ten million rows the last one reads 1.2 MB for that).
__global__ __launch_bounds__(256) void list_candidates_kernel(const uint64_t* mask, const uint64_t* present, uint64_t n_rows,
                                                              uint32_t* list, uint32_t* count) {
    __shared__ uint32_t wave_sum[4];
    const uint64_t n_words = (n_rows + 63) / 64, first = (uint64_t)blockIdx.x * 1024;
    uint32_t n = 0, before, total;
    for (uint64_t i = threadIdx.x; i < first; i += 256) n += __popcll(word_at(mask, present, i, n_rows));
    block_exclusive(n, wave_sum, &before);
    uint64_t words[4];
    n = 0;
    for (int j = 0; j < 4; ++j) {
        const uint64_t i = first + threadIdx.x * 4 + j;
        words[j] = i < n_words ? word_at(mask, present, i, n_rows) : 0;
        n += __popcll(words[j]);
    }
    uint32_t at = before + block_exclusive(n, wave_sum, &total);
    for (int j = 0; j < 4; ++j)
        for (uint64_t w = words[j]; w; w &= w - 1)
            list[at++] = (uint32_t)((first + threadIdx.x * 4 + j) * 64 + __builtin_ctzll(w));
    if (blockIdx.x == gridDim.x - 1 && !threadIdx.x) *count = before + total;
}

// A query in the table's type, its factor, and the place of its click; one workgroup per query.
template <typename E, typename Q>
__global__ __launch_bounds__(256) void pack_queries_kernel(XentArgs a, const Q* queries, uint64_t stride, const uint32_t* targets,
                                                           float scale, uint32_t* click, float* qscale) {
    __shared__ float sums[4];
    const uint32_t q = blockIdx.x;
    E* out = static_cast<E*>(const_cast<void*>(a.q)) + (uint64_t)q * a.kp;
    float sq = 0;
    for (uint32_t k = threadIdx.x; k < a.kp; k += 256) {
        const E e = from_f32<E>(k < a.t.dim ? to_f32(queries[q * stride + k]) : 0.0f);
        sq = __builtin_fmaf(to_f32(e), to_f32(e), sq);
        out[k] = e;
    }
    sq = wave_sum(sq);
    if (!(threadIdx.x & 63)) sums[threadIdx.x >> 6] = sq;
    __syncthreads();
    if (threadIdx.x) return;
    const float norm = __builtin_sqrtf(sums[0] + sums[1] + sums[2] + sums[3]);
    qscale[q] = !a.norms ? scale : norm > 0 ? scale / norm : 0.0f;
    const uint32_t id = targets[q], row = id - a.t.first_id;
    uint32_t place = id >= a.t.first_id && row < a.t.n_rows ? row : NONE;
    if (a.list && place != NONE) {
        uint32_t lo = 0, hi = *a.count;  // the first candidate that is not before the row
        while (lo < hi) {
            const uint32_t mid = (lo + hi) / 2;
            if (a.list[mid] < row)
                lo = mid + 1;
            else
                hi = mid;
        }
        place = lo < *a.count && a.list[lo] == row ? lo : NONE;
    }
    click[q] = place;
}

// ---- products -----------------------------------------------------------------------------

// A tile of 64 x 64 f32 sums by 256 threads, 4 x 4 each: sum over k of a(k, m) b(k, n).
template <typename A, typename B>
__device__ __forceinline__ void tile_product(A&& a, B&& b, uint32_t depth, float (&acc)[4][4]) {
    __shared__ float sa[16][64], sb[16][64];
    const uint32_t t = threadIdx.x, tm = t >> 4, tn = t & 15;
    for (uint32_t k0 = 0; k0 < depth; k0 += 16) {
        __syncthreads();
        for (uint32_t i = t; i < 1024; i += 256) {
            const uint32_t m = i >> 4, k = i & 15;
            sa[k][m] = k0 + k < depth ? a(k0 + k, m) : 0.0f;
            sb[k][m] = k0 + k < depth ? b(k0 + k, m) : 0.0f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 16; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = __builtin_fmaf(sa[k][tm * 4 + i], sb[k][tn * 4 + j], acc[i][j]);
    }
}

// Logit of the candidate at `place` for query q from their product.
__device__ __forceinline__ float logit(const XentArgs& a, uint32_t q, uint32_t place, float product) {
    float z = product * a.qscale[q];
    if (a.norms) {
        const float n = a.norms[row_at(a, place)];
        z = n > 0 ? z / n : 0.0f;
    }
    return z;
}

// Products of the 64 candidates from `first` (rows of the tile) with the 64 queries from q0 (columns).
template <typename E>
__device__ __forceinline__ void scores(const XentArgs& a, uint32_t first, uint32_t n, uint32_t q0, float (&acc)[4][4]) {
    const E* rows = static_cast<const E*>(a.t.rows);
    const E* q = static_cast<const E*>(a.q);
    tile_product([&](uint32_t k, uint32_t m) { return first + m < n ? to_f32(rows[row_at(a, first + m) * a.t.stride + k]) : 0.0f; },
                 [&](uint32_t k, uint32_t m) { return q0 + m < a.n_q ? to_f32(q[(uint64_t)(q0 + m) * a.kp + k]) : 0.0f; },
                 a.t.dim, acc);
}

template <typename E>
__global__ __launch_bounds__(256) void loss_kernel(XentArgs a) {
    __shared__ float sm[16][64], sl[16][64];
    const uint32_t t = threadIdx.x, tm = t >> 4, tn = t & 15, q0 = blockIdx.y * 64;
    const uint32_t n = candidates(a);
    float m[4], l[4] = {};
#pragma unroll
    for (int j = 0; j < 4; ++j) m[j] = -__builtin_inff();
    for (uint32_t first = blockIdx.x * 64; first < n; first += gridDim.x * 64) {
        float acc[4][4] = {};
        scores<E>(a, first, n, q0, acc);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t q = q0 + tn * 4 + j;
            if (q >= a.n_q) continue;
            const uint32_t click = a.click[q];
            for (int i = 0; i < 4; ++i) {
                const uint32_t place = first + tm * 4 + i;
                if (place >= n) continue;
                const float z = logit(a, q, place, acc[i][j]);
                if (place == click) {
                    a.click_z[q] = z;
                    continue;
                }
                const float top = __builtin_fmaxf(m[j], z), ref = top == -__builtin_inff() ? 0.0f : top;
                l[j] = l[j] * __expf(m[j] - ref) + __expf(z - ref);
                m[j] = top;
            }
        }
    }
    for (int j = 0; j < 4; ++j) {
        sm[tm][tn * 4 + j] = m[j];
        sl[tm][tn * 4 + j] = l[j];
    }
    __syncthreads();
    if (t >= 64 || q0 + t >= a.n_q) return;
    float top = -__builtin_inff(), sum = 0;
    for (int i = 0; i < 16; ++i) top = __builtin_fmaxf(top, sm[i][t]);
    for (int i = 0; i < 16; ++i) sum += sl[i][t] * __expf(sm[i][t] - (top == -__builtin_inff() ? 0.0f : top));
    a.part_m[(uint64_t)blockIdx.x * a.n_q + q0 + t] = top;
    a.part_l[(uint64_t)blockIdx.x * a.n_q + q0 + t] = sum;
}

// A query's parts joined, in 64 bits (one thread's worth of work per query); one workgroup per query.
__global__ __launch_bounds__(256) void join_loss_kernel(XentArgs a, float* loss, float* lse) {
    __shared__ float sm[256];
    __shared__ double sl[256];
    const uint32_t q = blockIdx.x, t = threadIdx.x;
    float top = -__builtin_inff();
    for (uint32_t s = t; s < a.splits; s += 256) top = __builtin_fmaxf(top, a.part_m[(uint64_t)s * a.n_q + q]);
    sm[t] = top;
    __syncthreads();
    for (int d = 128; d; d /= 2) {
        if (t < d) sm[t] = __builtin_fmaxf(sm[t], sm[t + d]);
        __syncthreads();
    }
    top = sm[0];
    const float ref = top == -__builtin_inff() ? 0.0f : top;
    double sum = 0;
    for (uint32_t s = t; s < a.splits; s += 256) {
        const uint64_t at = (uint64_t)s * a.n_q + q;
        sum += (double)a.part_l[at] * exp((double)a.part_m[at] - ref);
    }
    sl[t] = sum;
    __syncthreads();
    for (int d = 128; d; d /= 2) {
        if (t < d) sl[t] += sl[t + d];
        __syncthreads();
    }
    if (t) return;
    const double rest = ref + log(sl[0]);  // -inf: no other candidate
    if (a.click[q] == NONE) {
        loss[q] = 0.0f;
        lse[q] = (float)rest;
        return;
    }
    const double z = a.click_z[q], d = rest - z;
    loss[q] = (float)(d > 0 ? d + log1p(exp(-d)) : log1p(exp(d)));
    lse[q] = (float)(d > 0 ? rest + log1p(exp(-d)) : z + log1p(exp(d)));
}

// ---- gradients ----------------------------------------------------------------------------

template <typename E>
__global__ __launch_bounds__(256) void weights_kernel(XentArgs a) {
    const uint32_t t = threadIdx.x, tm = t >> 4, tn = t & 15, q0 = blockIdx.y * 64;
    const uint32_t n = candidates(a), first = a.piece_begin + blockIdx.x * 64;
    if (first >= n) return;
    float acc[4][4] = {};
    scores<E>(a, first, n, q0, acc);
    for (int i = 0; i < 4; ++i) {
        const uint32_t place = first + tm * 4 + i;
        if (place >= n) continue;
        for (int j = 0; j < 4; ++j) {
            const uint32_t q = q0 + tn * 4 + j;
            if (q >= a.n_q) continue;
            const uint32_t click = a.click[q];
            const float z = logit(a, q, place, acc[i][j]);
            float g = place == click ? expm1f(-a.loss[q]) : __expf(z - a.lse[q]);
            g *= (a.grad_loss ? a.grad_loss[q] : 1.0f) * a.qscale[q];
            if (a.norms) {
                const float norm = a.norms[row_at(a, place)];
                g = norm > 0 ? g / norm : 0.0f;
            }
            a.g[(uint64_t)(place - a.piece_begin) * a.n_q + q] = click == NONE ? 0.0f : g;
        }
    }
}

template <typename E>
__global__ __launch_bounds__(256) void row_grads_kernel(XentArgs a) {
    const uint32_t t = threadIdx.x, tm = t >> 4, tn = t & 15, d0 = blockIdx.y * 64;
    const uint32_t n = candidates(a), first = a.piece_begin + blockIdx.x * 64;
    if (first >= n) return;
    const E* q = static_cast<const E*>(a.q);
    float acc[4][4] = {};
    tile_product([&](uint32_t k, uint32_t m) { return first + m < n ? a.g[(uint64_t)(first + m - a.piece_begin) * a.n_q + k] : 0.0f; },
                 [&](uint32_t k, uint32_t m) { return d0 + m < a.t.dim ? to_f32(q[(uint64_t)k * a.kp + d0 + m]) : 0.0f; }, a.n_q, acc);
    E* out = static_cast<E*>(a.grad_rows);
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const uint32_t place = first + tm * 4 + i, d = d0 + tn * 4 + j;
            if (place < n && d < a.t.dim) out[row_at(a, place) * a.grad_row_stride + d] = from_f32<E>(acc[i][j]);
        }
}

// dqueries over one share of a piece's candidates.
template <typename E>
__global__ __launch_bounds__(256) void query_grads_kernel(XentArgs a) {
    const uint32_t t = threadIdx.x, tm = t >> 4, tn = t & 15, d0 = blockIdx.y * 64, q0 = blockIdx.z * 64;
    const uint32_t n = min(candidates(a), a.piece_begin + a.piece_rows);
    const uint32_t share = (a.piece_rows + a.splits - 1) / a.splits;
    const uint32_t begin = min(a.piece_begin + blockIdx.x * share, n), end = min(begin + share, n);
    const E* rows = static_cast<const E*>(a.t.rows);
    float acc[4][4] = {};
    tile_product([&](uint32_t k, uint32_t m) { return q0 + m < a.n_q ? a.g[(uint64_t)(begin + k - a.piece_begin) * a.n_q + q0 + m] : 0.0f; },
                 [&](uint32_t k, uint32_t m) { return d0 + m < a.t.dim ? to_f32(rows[row_at(a, begin + k) * a.t.stride + d0 + m]) : 0.0f; },
                 end - begin, acc);
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const uint32_t q = q0 + tm * 4 + i, d = d0 + tn * 4 + j;
            if (q >= a.n_q || d >= a.t.dim) continue;
            float* p = a.part_q + ((uint64_t)blockIdx.x * a.n_q + q) * a.t.dim + d;
            *p = a.first_piece ? acc[i][j] : *p + acc[i][j];
        }
}

// The shares of a query's gradient joined, and taken through the query's length where logits are cosines; one
// workgroup per query.
template <typename E, typename O>
__global__ __launch_bounds__(256) void join_query_grads_kernel(XentArgs a, O* out, uint64_t out_stride) {
    __shared__ float sums[8];
    const uint32_t q = blockIdx.x;
    const E* query = static_cast<const E*>(a.q) + (uint64_t)q * a.kp;
    float* sum0 = a.part_q + (uint64_t)q * a.t.dim;
    float dot = 0, sq = 0;
    for (uint32_t d = threadIdx.x; d < a.t.dim; d += 256) {
        float sum = 0;
        for (uint32_t s = 0; s < a.splits; ++s) sum += a.part_q[((uint64_t)s * a.n_q + q) * a.t.dim + d];
        if (!a.norms) {
            out[q * out_stride + d] = from_f32<O>(sum);
            continue;
        }
        const float x = to_f32(query[d]);
        dot = __builtin_fmaf(sum, x, dot);
        sq = __builtin_fmaf(x, x, sq);
        sum0[d] = sum;
    }
    if (!a.norms) return;
    dot = wave_sum(dot);
    sq = wave_sum(sq);
    if (!(threadIdx.x & 63)) {
        sums[threadIdx.x >> 6] = dot;
        sums[4 + (threadIdx.x >> 6)] = sq;
    }
    __syncthreads();
    dot = sums[0] + sums[1] + sums[2] + sums[3];
    sq = sums[4] + sums[5] + sums[6] + sums[7];
    const float along = sq > 0 ? dot / sq : 0.0f;
    for (uint32_t d = threadIdx.x; d < a.t.dim; d += 256) out[q * out_stride + d] = from_f32<O>(sum0[d] - along * to_f32(query[d]));
}

// Rows that are no candidates have gradient zero (`all`: every row, where there is no query).
template <typename E>
__global__ __launch_bounds__(256) void clear_rows_kernel(const uint64_t* mask, const uint64_t* present, bool all, uint64_t n_rows,
                                                         uint32_t dim, E* out, uint64_t stride) {
    for (uint64_t r = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < n_rows; r += (uint64_t)gridDim.x * 4) {
        if (!all && word_at(mask, present, r >> 6, n_rows) >> (r & 63) & 1) continue;
        for (uint32_t d = threadIdx.x & 63; d < dim; d += 64) out[r * stride + d] = from_f32<E>(0.0f);
    }
}

// ---- host side ----------------------------------------------------------------------------

constexpr uint64_t PIECE_BYTES = 256u << 20;  // of the gradient weights that are held at a time

struct Plan {
    uint32_t kp, loss_splits, grad_splits;
    uint64_t piece_rows;
};

Plan plan_for(uint32_t n_q, uint64_t n_rows, uint32_t dim, int32_t dtype) {
    Plan p;
    p.kp = (dim + 63) / 64 * 64;
    p.loss_splits = (uint32_t)std::min<uint64_t>((n_rows + 63) / 64, 1024);
    p.piece_rows = std::min<uint64_t>(std::max<uint64_t>(PIECE_BYTES / 4 / n_q / 64 * 64, 64), (n_rows + 63) / 64 * 64);
    p.grad_splits = (uint32_t)std::min<uint64_t>((p.piece_rows + 63) / 64, 16);
    return p;
}

struct Buffers {
    uint32_t *list, *count, *click;
    float *qscale, *part_m, *part_l, *click_z, *g, *part_q;
    void* q;
    uint64_t bytes;
};
Buffers carve(void* workspace, const Plan& p, uint32_t n_q, uint64_t n_rows, uint32_t dim, int32_t dtype) {
    Carver w(workspace);
    Buffers b;
    b.list = w.take<uint32_t>(n_rows);
    b.count = w.take<uint32_t>(1);
    b.click = w.take<uint32_t>(n_q);
    b.qscale = w.take<float>(n_q);
    b.click_z = w.take<float>(n_q);
    b.q = w.take<char>((uint64_t)n_q * p.kp * (dtype == VS_F32 ? 4 : 2));
    b.part_m = w.take<float>((uint64_t)p.loss_splits * n_q);
    b.part_l = w.take<float>((uint64_t)p.loss_splits * n_q);
    b.g = w.take<float>(p.piece_rows * n_q);
    b.part_q = w.take<float>((uint64_t)p.grad_splits * n_q * dim);
    b.bytes = w.at() - (char*)workspace;
    return b;
}

XentArgs prepare(const Xent& x, const Plan& p, const Buffers& b, hipStream_t stream) {
    XentArgs a{};
    a.t = x.t;
    a.norms = x.norms;
    a.q = b.q;
    a.kp = p.kp;
    a.n_q = x.n_q;
    a.click = b.click;
    a.qscale = b.qscale;
    a.part_m = b.part_m;
    a.part_l = b.part_l;
    a.click_z = b.click_z;
    a.g = b.g;
    a.part_q = b.part_q;
    if (x.mask || x.t.present) {
        a.list = b.list;
        a.count = b.count;
        const uint64_t n_words = (x.t.n_rows + 63) / 64;
        list_candidates_kernel<<<(uint32_t)((n_words + 1023) / 1024), 256, 0, stream>>>(x.mask, x.t.present, x.t.n_rows, b.list, b.count);
    }
    if (x.t.dtype == VS_F32)
        pack_queries_kernel<float, float><<<x.n_q, 256, 0, stream>>>(a, (const float*)x.queries, x.query_stride, x.targets, x.scale, b.click, b.qscale);
    else if (x.queries_f32)
        pack_queries_kernel<bf16, float><<<x.n_q, 256, 0, stream>>>(a, (const float*)x.queries, x.query_stride, x.targets, x.scale, b.click, b.qscale);
    else
        pack_queries_kernel<bf16, bf16><<<x.n_q, 256, 0, stream>>>(a, (const bf16*)x.queries, x.query_stride, x.targets, x.scale, b.click, b.qscale);
    return a;
}

template <typename E>
void run_grads(XentArgs a, const Plan& p, bool rows_too, hipStream_t stream) {
    const uint32_t qb = (a.n_q + 63) / 64, db = (a.t.dim + 63) / 64;
    for (uint64_t begin = 0; begin < a.t.n_rows; begin += p.piece_rows) {
        a.piece_begin = (uint32_t)begin;
        a.piece_rows = (uint32_t)std::min<uint64_t>(p.piece_rows, a.t.n_rows - begin);
        a.first_piece = !begin;
        const uint32_t tiles = (a.piece_rows + 63) / 64;
        weights_kernel<E><<<dim3(tiles, qb), 256, 0, stream>>>(a);
        if (rows_too) row_grads_kernel<E><<<dim3(tiles, db), 256, 0, stream>>>(a);
        if (a.part_q) query_grads_kernel<E><<<dim3(a.splits, db, qb), 256, 0, stream>>>(a);
    }
}

void clear_rows(const Xent& x, void* grad_rows, uint64_t stride, bool all, hipStream_t stream) {
    const uint32_t grid = (uint32_t)std::min<uint64_t>((x.t.n_rows + 3) / 4, 1u << 16);
    if (x.t.dtype == VS_F32)
        clear_rows_kernel<<<grid, 256, 0, stream>>>(x.mask, x.t.present, all, x.t.n_rows, x.t.dim, (float*)grad_rows, stride);
    else
        clear_rows_kernel<<<grid, 256, 0, stream>>>(x.mask, x.t.present, all, x.t.n_rows, x.t.dim, (bf16*)grad_rows, stride);
}

}  // namespace

uint64_t xent_workspace_bytes(uint32_t n_q, uint64_t n_rows, uint32_t dim, int32_t dtype) {
    return carve(nullptr, plan_for(n_q, n_rows, dim, dtype), n_q, n_rows, dim, dtype).bytes + 256;
}

hipError_t launch_xent(const Xent& x, void* workspace, float* loss, float* lse, hipStream_t stream) {
    const Plan p = plan_for(x.n_q, x.t.n_rows, x.t.dim, x.t.dtype);
    XentArgs a = prepare(x, p, carve(workspace, p, x.n_q, x.t.n_rows, x.t.dim, x.t.dtype), stream);
    a.splits = p.loss_splits;
    const dim3 grid(a.splits, (x.n_q + 63) / 64);
    if (x.t.dtype == VS_F32)
        loss_kernel<float><<<grid, 256, 0, stream>>>(a);
    else
        loss_kernel<bf16><<<grid, 256, 0, stream>>>(a);
    join_loss_kernel<<<x.n_q, 256, 0, stream>>>(a, loss, lse);
    return hipGetLastError();
}

hipError_t launch_xent_grad(const Xent& x, const float* loss, const float* lse, const float* grad_loss, void* workspace,
                            void* grad_queries, bool grad_queries_f32, uint64_t grad_query_stride, void* grad_rows,
                            uint64_t grad_row_stride, hipStream_t stream) {
    if (!x.n_q) {
        if (grad_rows) clear_rows(x, grad_rows, grad_row_stride, true, stream);
        return hipGetLastError();
    }
    const Plan p = plan_for(x.n_q, x.t.n_rows, x.t.dim, x.t.dtype);
    XentArgs a = prepare(x, p, carve(workspace, p, x.n_q, x.t.n_rows, x.t.dim, x.t.dtype), stream);
    a.splits = p.grad_splits;
    a.loss = loss;
    a.lse = lse;
    a.grad_loss = grad_loss;
    a.grad_rows = grad_rows;
    a.grad_row_stride = grad_row_stride;
    if (!grad_queries) a.part_q = nullptr;
    if (grad_rows && a.list) clear_rows(x, grad_rows, grad_row_stride, false, stream);
    if (x.t.dtype == VS_F32)
        run_grads<float>(a, p, grad_rows != nullptr, stream);
    else
        run_grads<bf16>(a, p, grad_rows != nullptr, stream);
    if (grad_queries) {
        if (x.t.dtype == VS_F32)
            join_query_grads_kernel<float, float><<<x.n_q, 256, 0, stream>>>(a, (float*)grad_queries, grad_query_stride);
        else if (grad_queries_f32)
            join_query_grads_kernel<bf16, float><<<x.n_q, 256, 0, stream>>>(a, (float*)grad_queries, grad_query_stride);
        else
            join_query_grads_kernel<bf16, bf16><<<x.n_q, 256, 0, stream>>>(a, (bf16*)grad_queries, grad_query_stride);
    }
    return hipGetLastError();
}

}  // namespace learn
}  // namespace vs
