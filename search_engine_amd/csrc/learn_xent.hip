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
//
// Four products on the bf16 matrix cores (learn_mma.h) carry it: rows x queries for the loss, the same again for the
// weights G, and G with the queries and with the rows for the gradients. Up to four queries make their logits by plain products,
// both times. G is made for a piece of the rows at a time and
// read twice before the next piece takes its place. Rows that are not whole 16-byte chunks at multiples of 16 bytes are
// copied to such, piece by piece, first.
#include "../../include/vs_abi.h"
#include "learn_kernels.h"
#include "learn_mma.h"

#include <type_traits>

namespace vs {
namespace learn {
namespace {

constexpr uint32_t NONE = 0xFFFFFFFFu;
constexpr float LOG2E = 1.44269504088896340736f;
constexpr int TILE = 256;  // candidates of a tile
constexpr uint32_t NO_ROW = 0xF0000000u;  // behind every row, and no sum with a tile's rows wraps

struct XentArgs {
    Planes rows;            // of the candidates, or of the whole table with the list of candidates
    uint32_t place0;        // the candidate that is row 0 of `rows`
    uint64_t n_rows;        // candidates where there is no list
    const uint32_t* list;   // candidate rows, ascending; null = every row
    const uint32_t* count;  // of the list
    const float* norms;
    Planes q;               // queries, with the sign of the scale
    Planes qt;              // queries transposed
    uint32_t n_q, gq, dim;  // gq: n_q rounded up to 64
    const uint32_t* click;  // [n_q] place of the clicked row among the candidates, or NONE
    const float* qscale;    // [n_q] factor of a query's products, without its sign
    float sign;
    Steps grad_steps;
    const char* zeros;
    uint32_t piece_begin, piece_rows;
    bool first_piece;
    uint32_t across, splits;  // workgroups side by side (query or column tiles), and along the rows
    float *part_m, *part_l;   // [splits][n_q] of the loss, base 2
    // gradients
    const float *lse, *loss, *grad_loss;
    char* g;                  // [planes][piece][whole tiles of queries] bf16
    uint64_t g_plane;
    uint32_t g_stride, g_planes;
    float* click_rest;        // [n_q] what the queries' product does not see of the clicked row's weight
    char* spill;              // 16 bytes of every thread of a product, for what it has no place for
    void* grad_rows;
    uint64_t grad_row_stride;
    float* part_q;            // [splits][n_q][dim]
};

// What is read as the caller has it: by the loss of a few queries all of it, else the clicks.
struct Few {
    const void *rows, *queries;
    uint64_t stride, query_stride;
    const uint32_t* targets;
    const uint64_t *mask, *present;
    uint32_t first_id;
    float scale;
    uint32_t parts;  // of a word that waves take: 1, 2, 4 or 8
};

// (told to the compiler as one value for all lanes: the loops of the products run on it)
__device__ __forceinline__ uint32_t candidates(const XentArgs& a) {
    return uniform_u32(a.list ? *a.count : (uint32_t)a.n_rows);
}
__device__ __forceinline__ uint64_t row_at(const XentArgs& a, uint32_t place) { return a.list ? a.list[place] : place; }

// The dispatcher deals workgroups out to the eight XCDs in turn. Renumbered, an XCD's are neighbours: those that share a
// tile of rows, `across` of them, are on one XCD (or two), and its L2 holds the tile for all of them (dealt out as they come,
// the gradient of 256 queries from 250 thousand x 768 f32 fetched 3.8 GB, so 1.6).
__device__ __forceinline__ void place_of_workgroup(uint32_t across, uint32_t* a, uint32_t* along) {
    const uint32_t xcd = blockIdx.x & 7, n = xcd * (gridDim.x >> 3) + min(xcd, gridDim.x & 7) + (blockIdx.x >> 3);
    *a = n % across;
    *along = n / across;
}

// ---- candidates and queries ------------------------------------------------------------------

__device__ __forceinline__ uint64_t word_at(const uint64_t* mask, const uint64_t* present, uint64_t i, uint64_t n_rows) {
    uint64_t w = mask ? mask[i] : ~0ull;
    if (present) w &= present[i];
    const uint64_t left = n_rows - i * 64;
    return left < 64 ? w & ((1ull << left) - 1) : w;
}

__device__ __forceinline__ bool clicked_candidate(const Few& f, uint32_t q, uint64_t n_rows) {
    const uint32_t id = f.targets[q], row = id - f.first_id;
    return id >= f.first_id && row < n_rows && word_at(f.mask, f.present, row >> 6, n_rows) >> (row & 63) & 1;
}

// An element of a query as it is multiplied with rows of type E.
template <typename E, typename Q>
__device__ __forceinline__ float query_element(Q x) {
    return sizeof(E) == 2 ? __builtin_bit_cast(float, bf16_bits(to_f32(x)) << 16) : to_f32(x);
}

// The candidate rows in ascending order: 256 words of the masks per workgroup, which counts the words before its own by
// itself, or (`sums` given) adds up the counts that count_words_kernel has left for each 256 words. A wave writes a word's rows together, lane l the l-th
// bit's: a lane writing its own word's rows would touch a line of its own with each.
constexpr uint32_t LIST_WORDS = 256;
__global__ __launch_bounds__(256) void count_words_kernel(const uint64_t* mask, const uint64_t* present, uint64_t n_rows, uint32_t* sums) {
    __shared__ uint32_t wave_sum[4];
    const uint64_t i = (uint64_t)blockIdx.x * LIST_WORDS + threadIdx.x;
    uint32_t total;
    block_exclusive(i < (n_rows + 63) / 64 ? __popcll(word_at(mask, present, i, n_rows)) : 0, wave_sum, &total);
    if (!threadIdx.x) sums[blockIdx.x] = total;
}
__global__ __launch_bounds__(256) void list_candidates_kernel(const uint64_t* mask, const uint64_t* present, uint64_t n_rows,
                                                              const uint32_t* sums, uint32_t* list, uint32_t* count) {
    __shared__ uint32_t wave_sum[4];
    const uint64_t n_words = (n_rows + 63) / 64, first = (uint64_t)blockIdx.x * LIST_WORDS;
    uint32_t n = 0, before, total;
    if (sums)
        for (uint32_t i = threadIdx.x; i < blockIdx.x; i += 256) n += sums[i];
    else
        for (uint64_t i = threadIdx.x; i < first; i += 256) n += __popcll(word_at(mask, present, i, n_rows));
    block_exclusive(n, wave_sum, &before);
    const uint64_t i = first + threadIdx.x;
    const uint64_t word = i < n_words ? word_at(mask, present, i, n_rows) : 0;
    const uint32_t at = before + block_exclusive((uint32_t)__popcll(word), wave_sum, &total);
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t row0 = (uint32_t)(first + (threadIdx.x & ~63u)) * 64;  // of the wave's first word
    for (int k = 0; k < 64; ++k) {
        const uint64_t w = readlane_u64(word, k);
        const uint32_t to = (uint32_t)__builtin_amdgcn_readlane((int)at, k);
        if (w >> lane & 1) list[to + __popcll(w & ((1ull << lane) - 1))] = row0 + k * 64 + lane;
    }
    if (blockIdx.x == gridDim.x - 1 && !threadIdx.x) *count = before + total;
}

// Queries as planes (5 - 9 us: latency), [n_q][k] and, for gradients, transposed [dim][gq], by tiles of 64 x 64; the workgroups behind the
// tiles take four queries each: length, factor, and the place of the click. For gradients a query whose click is no
// candidate is zeros, whatever it holds (padding of a batch may hold anything): its weights are zero, and zero times what
// is no number would be none in every row's gradient.
template <typename Q, int P>
__global__ __launch_bounds__(256) void pack_queries_kernel(XentArgs a, Few f, uint32_t* click, float* qscale, uint32_t* zeros,
                                                           bool gradients) {
    __shared__ uint16_t t[P][64][72];  // [column][query], eight queries more than there are: rows stay 16-byte aligned
    const Q* const queries = static_cast<const Q*>(f.queries);
    const uint64_t stride = f.query_stride;
    const uint32_t n_tiles = a.gq / 64 * (a.q.chunks / 8);
    if (!blockIdx.x && threadIdx.x < 64) zeros[threadIdx.x] = 0;
    if (blockIdx.x < n_tiles) {
        const uint32_t q0 = blockIdx.x % (a.gq / 64) * 64, d0 = blockIdx.x / (a.gq / 64) * 64;
#pragma unroll
        for (uint32_t k = 0; k < 512; k += 256) {
            const uint32_t i = k + threadIdx.x, q = q0 + i / 8, d = d0 + i % 8 * 8;
            const bool in = q < a.n_q && (!gradients || clicked_candidate(f, q, a.n_rows));
            Pack<uint16_t, 8> part[3];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const Split s = split(in && d + j < a.dim ? to_f32(queries[q * stride + d + j]) : 0.0f);
                part[0].e[j] = s.h;
                part[1].e[j] = s.m;
                part[2].e[j] = s.l;
            }
#pragma unroll
            for (int p = 0; p < P; ++p) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    t[p][i % 8 * 8 + j][i / 8] = part[p].e[j];
                    part[p].e[j] ^= a.sign < 0 ? 0x8000 : 0;
                }
                if (q < a.n_q)
                    store_pack<uint16_t, 8>(reinterpret_cast<uint16_t*>(const_cast<char*>(a.q.base) + p * a.q.plane + q * (uint64_t)a.q.stride) + d, part[p]);
            }
        }
        if (!gradients) return;
        __syncthreads();
#pragma unroll
        for (uint32_t k = 0; k < 512; k += 256) {
            const uint32_t i = k + threadIdx.x, d = d0 + i / 8, q = q0 + i % 8 * 8;
            if (d >= a.dim) continue;
#pragma unroll
            for (int p = 0; p < P; ++p)
                store_pack<uint16_t, 8>(reinterpret_cast<uint16_t*>(const_cast<char*>(a.qt.base) + p * a.qt.plane + d * (uint64_t)a.qt.stride) + q,
                                        load_pack<uint16_t, 8>(&t[p][i / 8][i % 8 * 8]));
        }
        return;
    }
    const uint32_t q = (blockIdx.x - n_tiles) * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (q >= a.n_q) return;
    double sq = 0;  // (64 bits: f32 holds no square of a vector longer than 2^64, or shorter than 2^-75)
    if (a.norms) {
        for (uint32_t d = lane; d < a.dim; d += 64) {
            const double x = query_element<std::conditional_t<P == 1, bf16, float>>(queries[q * stride + d]);
            sq += x * x;
        }
        sq = wave_sum(sq);
    }
    if (lane) return;
    const float norm = (float)sqrt(sq), size = __builtin_fabsf(f.scale);
    qscale[q] = !a.norms ? size : norm > 0 ? size / norm : 0.0f;
    const uint32_t row = f.targets[q] - f.first_id;
    uint32_t place = clicked_candidate(f, q, a.n_rows) ? row : NONE;
    if (a.list && place != NONE) {
        uint32_t lo = 0, hi = *a.count;  // where the row stands in the list
        while (lo < hi) {
            const uint32_t mid = (lo + hi) / 2;
            if (a.list[mid] < row)
                lo = mid + 1;
            else
                hi = mid;
        }
        place = lo;
    }
    click[q] = place;
}

// A piece of the candidates as rows that start at multiples of 16 bytes, zeros from `dim` on: 16 bytes a thread (45 thousand
// x 383 f32: 23 us, 6.0 TB/s).
template <typename E>
__global__ __launch_bounds__(256) void pack_rows_kernel(XentArgs a, const E* table, uint64_t stride, char* out) {
    constexpr int V = 16 / sizeof(E);
    const uint32_t end = min(candidates(a), a.piece_begin + a.piece_rows);
    const uint64_t total = end > a.piece_begin ? (uint64_t)(end - a.piece_begin) * a.rows.chunks : 0;
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (uint64_t)gridDim.x * 256) {
        const uint32_t r = (uint32_t)(i / a.rows.chunks), d = (uint32_t)(i - (uint64_t)r * a.rows.chunks) * V;
        const E* from = table + row_at(a, a.piece_begin + r) * stride + d;
        store_pack<E, V>(reinterpret_cast<E*>(out + r * (uint64_t)a.rows.stride) + d, load_any<E, V>(from, d < a.dim ? a.dim - d : 0));
    }
}

// ---- products -----------------------------------------------------------------------------

// Tiles of candidates with one tile of queries: BQ queries by TILE candidates, `along` of `splits` workgroups. `done` is
// called with each tile's sums and its first place; the loads of the next tile's first step are under way meanwhile.
// LANES_ARE_QUERIES: a lane holds four candidates (rows of the product) of one query, else four queries of one candidate.
template <int BQ, bool LANES_ARE_QUERIES, bool LISTED>
struct Scores {
    static constexpr int WAVES_Q = BQ >= 256 ? 4 : BQ >= 128 ? 2 : 1;  // waves side by side along the queries
    static constexpr int WAVES_R = 8 / WAVES_Q;
    static constexpr int WQ = BQ / WAVES_Q / 16, WR = TILE / WAVES_R / 16;  // fragments of a wave
    static constexpr int TM = LANES_ARE_QUERIES ? WR : WQ, TN = LANES_ARE_QUERIES ? WQ : WR;
    static constexpr int T = TILE, Q_TILE = BQ, UNIT = TM < 4 ? TM : 4;  // (fragments of weights that go through LDS at a time)
    static constexpr bool SPLIT = false;
    using R = Rows<TILE, LISTED>;
    using Q = Rows<BQ>;
    // Beside the buffers: results on their way out (16 KiB) and numbers of each query and candidate.
    static constexpr int BUFFERS = buffers_of(R::BYTES + Q::BYTES, 16384 + 6144);
    static constexpr int LDS = BUFFERS * (R::BYTES + Q::BYTES);

    __device__ __forceinline__ static uint32_t wave_q() { return uniform_u32(threadIdx.x >> 6) % WAVES_Q; }
    __device__ __forceinline__ static uint32_t wave_r() { return uniform_u32(threadIdx.x >> 6) / WAVES_Q; }

    // STORES: done() returns whether it made at least so many stores.
    template <int STORES, typename F>
    __device__ __forceinline__ static void run(const XentArgs& a, uint32_t end, uint32_t q0, uint32_t along, char* lds, F&& done) {
        Planes rows = a.rows;
        rows.rows = end - a.place0;
        R r;
        Q q;
        r.init();
        q.init();
        q.aim(q0);
        const uint32_t tiles = (end - a.piece_begin + TILE - 1) / TILE;
        if (along >= tiles) return;
        const uint32_t steps = (a.rows.chunks + 7) / 8;
        // (the pairs of planes of a step. Where rows come through the list and results through LDS, a compiler that knows it
        // to be one keeps addresses in registers that the sums need, and spills in the loop: 1.6 times the time)
        const uint32_t planes = LISTED && !LANES_ARE_QUERIES ? afresh_uniform(1) : 1;
        const uint32_t base = a.piece_begin - a.place0;
        auto half_r = [&](uint32_t i) { return lds + i * (R::BYTES + Q::BYTES); };
        auto half_q = [&](uint32_t i) { return lds + i * (R::BYTES + Q::BYTES) + R::BYTES; };
        // The rows have furthest to come: theirs go first, behind a step's barrier into the buffer that it has freed; the
        // queries of that step follow in the next step's first phases. Loads go on behind the last tile, of zeros, so
        // that their number stays what the barriers count on.
        Cursor cr{0, 0, along}, cq{0, 0, along};
        r.peek(rows, base + along * TILE);
        r.aim(base + along * TILE);
        r.peek(rows, base + (along + a.splits) * TILE);
        auto load_rows = [&](uint32_t to) {
#pragma unroll
            for (int i = 0; i < R::LOADS; ++i) r.load(i, rows, cr.k, 0, a.zeros, half_r(to));
            if (!cr.advance(planes, steps, a.splits)) return;
            r.aim(cr.tile < tiles ? base + cr.tile * TILE : NO_ROW);
            r.peek(rows, cr.tile + a.splits < tiles ? base + (cr.tile + a.splits) * TILE : 0);
        };
        auto load_queries = [&](int i, uint32_t to) { q.load(i, a.q, cq.k, 0, a.zeros, half_q(to)); };
        auto load_all_queries = [&](uint32_t to) {
#pragma unroll
            for (int i = 0; i < Q::LOADS; ++i) load_queries(i, to);
            cq.advance(planes, steps, a.splits);
        };
        constexpr int BEHIND = (BUFFERS - 2) * (R::LOADS + Q::LOADS);
#pragma unroll
        for (int i = 0; i < BUFFERS - 1; ++i) {
            load_rows(i);
            load_all_queries(i);
        }
        step_barrier<BEHIND>();
        using E = Engine<std::conditional_t<LANES_ARE_QUERIES, R, Q>, std::conditional_t<LANES_ARE_QUERIES, Q, R>, TM, TN>;
        E e;
        e.m0 = LANES_ARE_QUERIES ? wave_r() * WR : wave_q() * WQ;
        e.n0 = LANES_ARE_QUERIES ? wave_q() * WQ : wave_r() * WR;
        e.ask(LANES_ARE_QUERIES ? half_r(0) : half_q(0), LANES_ARE_QUERIES ? half_q(0) : half_r(0), 0);
        load_rows(BUFFERS - 1);
        uint32_t at = 0;
        uint32_t early = 0, stored = 0;  // the queries to be loaded in this step are under way already; stores are
#pragma nounroll
        for (uint32_t tile = along; tile < tiles; tile += a.splits) {
            f32x4 acc[TM][TN] = {};
#pragma nounroll
            for (uint32_t s = 0; s < steps; ++s) {
                const uint32_t next = at + 1 == BUFFERS ? 0 : at + 1, last = at ? at - 1 : BUFFERS - 1;
                char *ar = half_r(at), *aq = half_q(at), *br = half_r(next), *bq = half_q(next);
                e.template step<BEHIND, STORES>(LANES_ARE_QUERIES ? ar : aq, LANES_ARE_QUERIES ? aq : ar, LANES_ARE_QUERIES ? br : bq,
                                                LANES_ARE_QUERIES ? bq : br, acc, stored, [&](int phase) {
                    if (phase < E::PHASES - 1) {
                        constexpr int EACH = (Q::LOADS + E::PHASES - 2) / (E::PHASES - 1);
                        if (BUFFERS == 2 && STORES && early) return;
#pragma unroll
                        for (int i = phase * EACH; i < min((phase + 1) * EACH, Q::LOADS); ++i) load_queries(i, last);
                        return;
                    }
                    if (!(BUFFERS == 2 && STORES && early)) cq.advance(planes, steps, a.splits);
                    load_rows(at);
                    if (BUFFERS > 2 || !STORES) return;
                    // two buffers, and the tile's end stores: what the step after next needs goes before that
                    early = afresh_uniform(s + 1 == steps);
                    if (early) load_all_queries(at);
                });
                stored = afresh_uniform(0);
                at = next;
            }
            stored = afresh_uniform(done(acc, a.piece_begin + tile * TILE));
        }
        __builtin_amdgcn_s_waitcnt(0x0F70);  // (the zeros have come: nothing writes LDS behind the workgroup's end)
    }
};

// f32 tables: tiles of 64 queries, as planes, by T candidates as they are in the table. Rows go by 32 k at a time (half a
// step) through three buffers, queries by 64 through two.
template <bool LANES_ARE_QUERIES, bool LISTED, int ROWS>
struct SplitScores {
    static constexpr int T = ROWS, Q_TILE = 64, UNIT = T == 128 ? 4 : 2;
    static constexpr bool SPLIT = true;
    static constexpr int WAVES_Q = T == 64 ? 2 : 1, WAVES_R = 8 / WAVES_Q, WQ = 4 / WAVES_Q, WR = T / WAVES_R / 16;
    static constexpr int TM = LANES_ARE_QUERIES ? WR : WQ, TN = LANES_ARE_QUERIES ? WQ : WR;
    using R = Rows<T, LISTED>;
    using Q = Rows<Q_TILE>;
    static constexpr int LDS = 3 * R::BYTES + 2 * 3 * Q::BYTES;

    __device__ __forceinline__ static uint32_t wave_q() { return uniform_u32(threadIdx.x >> 6) % WAVES_Q; }
    __device__ __forceinline__ static uint32_t wave_r() { return uniform_u32(threadIdx.x >> 6) / WAVES_Q; }

    // As in Scores.
    template <int STORES, typename F>
    __device__ __forceinline__ static void run(const XentArgs& a, uint32_t end, uint32_t q0, uint32_t along, char* lds, F&& done) {
        Planes rows = a.rows;
        rows.rows = end - a.place0;
        R r;
        Q q;
        r.init();
        q.init();
        q.aim(q0);
        const uint32_t tiles = (end - a.piece_begin + T - 1) / T;
        if (along >= tiles) return;
        const uint32_t steps = (a.rows.chunks + 15) / 16, base = a.piece_begin - a.place0;
        auto half_r = [&](uint32_t i) { return lds + i * R::BYTES; };
        auto half_q = [&](uint32_t i) { return lds + 3 * R::BYTES + i * 3 * Q::BYTES; };
        Cursor cr{0, 0, along}, cq{0, 0, along};
        r.peek(rows, base + along * T);
        r.aim(base + along * T);
        r.peek(rows, base + (along + a.splits) * T);
        auto load_rows = [&](uint32_t to) {
#pragma unroll
            for (int i = 0; i < R::LOADS; ++i) r.load(i, rows, cr.k, 0, a.zeros, half_r(to));
            if (!cr.advance(1, 2 * steps, a.splits)) return;
            r.aim(cr.tile < tiles ? base + cr.tile * T : NO_ROW);
            r.peek(rows, cr.tile + a.splits < tiles ? base + (cr.tile + a.splits) * T : 0);
        };
        auto load_queries = [&](uint32_t to) {
#pragma unroll
            for (int p = 0; p < 3; ++p) q.load(0, a.q, cq.k, p, a.zeros, half_q(to) + p * Q::BYTES);
            cq.advance(1, steps, a.splits);
        };
        // What a barrier waits for are the next half's rows, and behind a step's second half the next step's queries; what
        // was issued after those may be under way: the rows of the half after it, and before a second half the queries.
        load_queries(0);
        load_rows(0);
        load_rows(1);
        load_queries(1);
        load_rows(2);
        step_barrier<3 + 2 * R::LOADS>();
        SplitEngine<Q, R, WQ, WR, !LANES_ARE_QUERIES> e;
        e.p0 = wave_q() * WQ;
        e.x0 = wave_r() * WR;
        e.start(half_q(0), half_r(0));
        uint32_t at = 0, at_q = 0, stored = 0;
        auto wait = [&](auto behind) {
            if (STORES && stored)
                step_barrier<behind + STORES>();
            else
                step_barrier<behind>();
        };
#pragma nounroll
        for (uint32_t tile = along; tile < tiles; tile += a.splits) {
            f32x4 acc[TM][TN] = {}, small[TM][TN] = {};
#pragma nounroll
            for (uint32_t s = 0; s < steps; ++s) {
                const uint32_t second = at == 2 ? 0 : at + 1, third = second == 2 ? 0 : second + 1, next_q = at_q ^ 1;
                e.template half<0>([&] { wait(std::integral_constant<int, R::LOADS + 3>{}); }, half_q(at_q), half_r(second), 0, acc, small,
                                   [&] { load_rows(at); });
                e.template half<1>([&] { wait(std::integral_constant<int, R::LOADS>{}); }, half_q(next_q), half_r(third), 0, acc, small, [&] {
                    load_queries(at_q);
                    load_rows(second);
                });
                stored = afresh_uniform(0);
                at = third;
                at_q = next_q;
            }
#pragma unroll
            for (int m = 0; m < TM; ++m)
#pragma unroll
                for (int n = 0; n < TN; ++n) acc[m][n] += small[m][n];
            stored = afresh_uniform(done(acc, a.piece_begin + tile * T));
        }
        __builtin_amdgcn_s_waitcnt(0x0F70);  // (as in Scores)
    }
};

__device__ __forceinline__ float finite_or_zero(float m) { return m == -__builtin_inff() ? 0.0f : m; }
// What products are multiplied with in base 2. (A factor of zero would make a NaN of the -inf that stands for what is left out:
// this one's logits are zero too.)
__device__ __forceinline__ float base2(float scale) {
    const float s2 = scale * LOG2E;
    return s2 == 0 ? 1.4e-45f : s2;
}

// Per query the largest logit of a share of the candidates and the sum of the exponentials over it, the clicked row kept
// out. Bound by the products from 64 queries (bf16) or so on, by the rows' bytes below: 256 queries over 1M x 768 bf16 take
// 390 - 450 us (0.87 - 1.0 PFLOP/s, by the clock; a large library product reaches 1.5), 10 take 255 (6.0 TB/s); over 250
// thousand x 768 f32 256 take 580 (168 TFLOP/s in f32 products, 1.0 PFLOP/s of the six bf16 ones: the wave's splitting and the
// matrix cores take 45 % of the cycles each). Everything is in base 2 (logits times log2 e): an exponential is one
// instruction. A lane keeps the running largest product and the sum of its own candidates, in registers, for each of its
// queries; lanes, waves and shares are joined at the end.
template <typename S, bool NORMS>
__global__ __launch_bounds__(THREADS, 2) void loss_kernel(XentArgs a) {
    constexpr int BQ = S::Q_TILE;
    extern __shared__ __attribute__((aligned(128))) char lds[];
    __shared__ float inverse[S::T], sm[S::WAVES_R][BQ], sl[S::WAVES_R][BQ];
    const uint32_t lane = threadIdx.x & 63, group = lane >> 4;
    uint32_t tile_q, along;
    place_of_workgroup(a.across, &tile_q, &along);
    const uint32_t end = min(candidates(a), a.piece_begin + a.piece_rows);
    uint32_t click[S::TN];
    float s2[S::TN], m[S::TN], l[S::TN];
#pragma unroll
    for (int n = 0; n < S::TN; ++n) {
        const uint32_t q = tile_q * BQ + (S::wave_q() * S::WQ + n) * 16 + (lane & 15);
        click[n] = q < a.n_q ? a.click[q] : NONE;
        s2[n] = base2(q < a.n_q ? a.qscale[q] : 0.0f);
        m[n] = -__builtin_inff();
        l[n] = 0;
    }
    if (end > a.piece_begin)
        S::template run<0>(a, end, tile_q * BQ, along, lds, [&](f32x4 (&acc)[S::TM][S::TN], uint32_t first) {
            if constexpr (NORMS) {
                // (the barriers of the steps before the next tile's end let everybody have read them. Where it would be zero,
                // of a length of zero or infinity, the factor is not: it would make a NaN of the -inf of what is left out)
                if (threadIdx.x < S::T) {
                    const float x = first + threadIdx.x < end ? a.norms[row_at(a, first + threadIdx.x)] : 0.0f, over = 1.0f / x;
                    inverse[threadIdx.x] = x > 0 && over > 0 ? over : 1.4e-45f;
                }
                __syncthreads();
            }
            const uint32_t local = S::wave_r() * S::WR * 16 + group * 4;  // of the lane's candidates t * 16 + r
            // (multiplied where they are used: the products themselves stay in the matrix cores' registers)
            auto length = [&](int t) {
                if constexpr (NORMS) return *reinterpret_cast<const f32x4*>(inverse + local + t * 16);
                return f32x4{1, 1, 1, 1};
            };
            bool special = end - first < S::T;
#pragma unroll
            for (int n = 0; n < S::TN; ++n) special |= click[n] - first < S::T;
            if (__any(special)) {
                // a tile with a clicked row, or the last one: what does not belong to the sum is taken out of it
#pragma unroll
                for (int n = 0; n < S::TN; ++n) {
                    const uint32_t at = click[n] - first - local;
                    const int left = (int)min(end - first, (uint32_t)S::T) - (int)local;
#pragma unroll
                    for (int t = 0; t < S::TM; ++t)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const uint32_t i = t * 16 + r;
                            acc[t][n][r] = at == i || left <= (int)i ? -__builtin_inff() : acc[t][n][r];
                        }
                }
            }
#pragma unroll
            for (int n = 0; n < S::TN; ++n) {
                float x = -__builtin_inff();
#pragma unroll
                for (int t = 0; t < S::TM; ++t) {
                    const f32x4 z = NORMS ? acc[t][n] * length(t) : acc[t][n];
#pragma unroll
                    for (int r = 0; r < 4; ++r) x = __builtin_fmaxf(x, z[r]);
                }
                const float top = __builtin_fmaxf(m[n], x);  // (the factor is not negative)
                const float ref = finite_or_zero(top * s2[n]);
                float sum[4] = {l[n] * __builtin_amdgcn_exp2f(m[n] * s2[n] - ref), 0, 0, 0};
#pragma unroll
                for (int t = 0; t < S::TM; ++t) {
                    const f32x4 z = NORMS ? acc[t][n] * length(t) : acc[t][n];
#pragma unroll
                    for (int r = 0; r < 4; ++r) sum[r] += __builtin_amdgcn_exp2f(__builtin_fmaf(z[r], s2[n], -ref));
                }
                l[n] = (sum[0] + sum[1]) + (sum[2] + sum[3]);
                m[n] = top;
            }
            return false;
        });
    // lanes that hold other candidates of the same query, then waves, then what the pieces before this one left
#pragma unroll
    for (int n = 0; n < S::TN; ++n) {
#pragma unroll
        for (int d = 16; d < 64; d *= 2) {
            const float om = __shfl_xor(m[n], d), ol = __shfl_xor(l[n], d), top = __builtin_fmaxf(m[n], om), ref = finite_or_zero(top * s2[n]);
            l[n] = l[n] * __builtin_amdgcn_exp2f(m[n] * s2[n] - ref) + ol * __builtin_amdgcn_exp2f(om * s2[n] - ref);
            m[n] = top;
        }
        if (lane < 16) {
            sm[S::wave_r()][(S::wave_q() * S::WQ + n) * 16 + lane] = m[n];
            sl[S::wave_r()][(S::wave_q() * S::WQ + n) * 16 + lane] = l[n];
        }
    }
    __syncthreads();
    const uint32_t q = tile_q * BQ + threadIdx.x;
    if (threadIdx.x >= BQ || q >= a.n_q) return;
    const uint64_t to = (uint64_t)along * a.n_q + q;
    float top = a.first_piece ? -__builtin_inff() : a.part_m[to], sum = a.first_piece ? 0.0f : a.part_l[to];
    const float before = top, factor = base2(a.qscale[q]);
    for (int w = 0; w < S::WAVES_R; ++w) top = __builtin_fmaxf(top, sm[w][threadIdx.x]);
    const float ref = finite_or_zero(top * factor);
    sum *= __builtin_amdgcn_exp2f(before * factor - ref);
    for (int w = 0; w < S::WAVES_R; ++w) sum += sl[w][threadIdx.x] * __builtin_amdgcn_exp2f(sm[w][threadIdx.x] * factor - ref);
    a.part_m[to] = top;
    a.part_l[to] = sum;
}

// Up to four queries: bound by the rows' bytes (one over 1M x 768 bf16: 243 us, 6.3 TB/s), so plain f32 products, straight from
// the table. The loss and the weights of the gradients share them, bit for bit: of a document that has nearly all of the
// probability, what its logit is off by is in lse and in its weight, and cancels only if it is the same.
template <typename E, typename Q, int V, int NQ, bool NORMS>
struct FewScores {
    static constexpr int U = NQ == 1 ? 8 : 4;  // candidates that a wave takes at a time, their loads in flight together
    uint32_t chunks, padded;                   // (a last, broken piece: see Piece)
    float* query;                              // [NQ][padded], as they are multiplied, with the sign of the scale
    float scale;                               // of the lane's query, lane % NQ: the logit of a product

    // By the whole workgroup of 256.
    __device__ __forceinline__ void init(const XentArgs& a, const Few& f, char* lds, double* sums /* 4, LDS */) {
        const uint32_t lane = threadIdx.x & 63, wave = uniform_u32(threadIdx.x >> 6);
        chunks = (a.dim + V - 1) / V;
        padded = chunks * V;
        query = reinterpret_cast<float*>(lds);
        scale = 0;
        const Q* queries = static_cast<const Q*>(f.queries);
        for (int q = 0; q < NQ; ++q) {
            double sq = 0;  // (as in pack_queries_kernel)
            for (uint32_t d = threadIdx.x; d < padded; d += 256) {
                const Piece<V> piece(d / V, a.dim);
                const uint32_t from = piece.col + d % V;
                const float x = d % V >= piece.skip && from < a.dim ? query_element<E>(queries[q * f.query_stride + from]) : 0.0f;
                query[q * padded + d] = f.scale < 0 ? -x : x;
                if constexpr (NORMS) sq += (double)x * x;
            }
            float its_scale = __builtin_fabsf(f.scale);
            if constexpr (NORMS) {
                sq = wave_sum(sq);
                __syncthreads();
                if (!lane) sums[wave] = sq;
                __syncthreads();
                const float norm = (float)sqrt(sums[0] + sums[1] + sums[2] + sums[3]);
                its_scale = norm > 0 ? its_scale / norm : 0.0f;
            }
            if (lane % NQ == (uint32_t)q) scale = its_scale;
        }
        __syncthreads();
    }
    // Lane u NQ + q gets candidate u's product with query q, and its row (cosines: over the row's length, and that).
    __device__ __forceinline__ float products(const XentArgs& a, const Few& f, const uint32_t (&row)[U], uint32_t* its_row, float* length) const {
        const uint32_t lane = threadIdx.x & 63;
        const E* const table = static_cast<const E*>(f.rows);
        float acc[U][NQ] = {};
        for (uint32_t c = lane; c < chunks; c += 64) {
            Pack<E, V> x[U];
#pragma unroll
            for (int u = 0; u < U; ++u) x[u] = load_piece_once<E, V>(table + (uint64_t)row[u] * f.stride, Piece<V>(c, a.dim), a.dim);
#pragma unroll
            for (int q = 0; q < NQ; ++q) {
                const Pack<float, V> y = load_pack<float, V>(query + q * padded + c * V);
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int v = 0; v < V; ++v) acc[u][q] = __builtin_fmaf(to_f32(x[u].e[v]), y.e[v], acc[u][q]);
            }
        }
        float z = 0;
        uint32_t r = row[0];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int q = 0; q < NQ; ++q) {
                const float sum = wave_sum(acc[u][q]);
                if (lane == (uint32_t)(u * NQ + q)) {
                    z = sum;
                    r = row[u];
                }
            }
        *its_row = r;
        if constexpr (NORMS) {
            *length = a.norms[r];
            z = *length == 0 ? 0.0f : z / *length;  // (a row that holds a NaN has no length, and no logit)
        }
        return z;
    }
};

// The loss, under the masks themselves, with nothing laid out before. A wave takes the words of the masks in turn, and of each
// word's candidates U at a time; the lane of each (candidate, query) keeps the running largest and sum of its logits.
template <typename E, typename Q, int V, int NQ, bool NORMS>
__global__ __launch_bounds__(256) void loss_few_kernel(XentArgs a, Few f, float* qscale) {
    using S = FewScores<E, Q, V, NQ, NORMS>;
    constexpr int U = S::U;
    extern __shared__ __attribute__((aligned(128))) char lds[];
    __shared__ float sm[4][64], sl[4][64];
    __shared__ double sums[4];
    const uint32_t lane = threadIdx.x & 63, wave = uniform_u32(threadIdx.x >> 6), mine = lane % NQ;
    S scores;
    scores.init(a, f, lds, sums);
    const float factor = base2(scores.scale);
    if (!blockIdx.x && threadIdx.x < NQ) qscale[threadIdx.x] = scores.scale;
    const uint32_t click = f.targets[mine] < f.first_id ? NONE : f.targets[mine] - f.first_id;
    float m = -__builtin_inff(), l = 0;
    const uint32_t n_units = (uint32_t)((a.n_rows + 63) / 64) * f.parts, size = 64 / f.parts;
    for (uint32_t i = blockIdx.x * 4 + wave; i < n_units; i += gridDim.x * 4) {
        const uint32_t w = i / f.parts, part = i % f.parts;
        uint64_t bits = uniform_u64(word_at(f.mask, f.present, w, a.n_rows));
        bits = bits >> (part * size) << (64 - size) >> (64 - size) << (part * size);
        while (bits) {
            uint32_t row[U];
            uint32_t n = 0;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                // (a place without a candidate repeats the last one's row, and its sum is not looked at)
                row[u] = bits ? w * 64 + (uint32_t)__builtin_ctzll(bits) : row[u ? u - 1 : 0];
                n += bits != 0;
                bits &= bits - 1;
            }
            uint32_t r;
            float length;
            const float z = scores.products(a, f, row, &r, &length);
            if (lane < n * NQ && r != click) {
                // (an fma: of a logit of hundreds the rounding alone would show in the exponential)
                const float top = __builtin_fmaxf(m, z), ref = finite_or_zero(top * factor);
                l = l * __builtin_amdgcn_exp2f(m * factor - ref) + __builtin_amdgcn_exp2f(__builtin_fmaf(z, factor, -ref));
                m = top;
            }
        }
    }
    sm[wave][lane] = m;
    sl[wave][lane] = l;
    __syncthreads();
    if (threadIdx.x >= NQ) return;
    float top = -__builtin_inff(), sum = 0;
    for (int w = 0; w < 4; ++w)
        for (int u = 0; u < U; ++u) top = __builtin_fmaxf(top, sm[w][u * NQ + threadIdx.x]);
    const float ref = finite_or_zero(top * factor);
    for (int w = 0; w < 4; ++w)
        for (int u = 0; u < U; ++u) sum += sl[w][u * NQ + threadIdx.x] * __builtin_amdgcn_exp2f(sm[w][u * NQ + threadIdx.x] * factor - ref);
    a.part_m[(uint64_t)blockIdx.x * NQ + threadIdx.x] = top;
    a.part_l[(uint64_t)blockIdx.x * NQ + threadIdx.x] = sum;
}

// A query's shares joined, in 64 bits; a workgroup per query: 5 - 10 us, two trips to memory one behind the other. The clicked
// row's logit is made here, in 64 bits: its error is that of a loss near zero, while those of the others' mostly cancel in
// their sum.
template <typename E, typename Q>
__global__ __launch_bounds__(256) void join_loss_kernel(XentArgs a, Few f, float* loss, float* lse) {
    __shared__ float tops[4];
    __shared__ double sums[4][3];
    const uint32_t q = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const bool clicked = clicked_candidate(f, q, a.n_rows);
    const uint32_t click = clicked ? f.targets[q] - f.first_id : 0;
    double dot = 0, sq = 0;
    if (clicked) {
        const E* const row = static_cast<const E*>(f.rows) + click * f.stride;
        const Q* const query = static_cast<const Q*>(f.queries) + q * f.query_stride;
#pragma unroll 4
        for (uint32_t d = threadIdx.x; d < a.dim; d += 256) {
            const double x = query_element<E>(query[d]);
            dot += x * to_f32(row[d]);
            sq += x * x;
        }
    }
    float top = -__builtin_inff();
    for (uint32_t s = threadIdx.x; s < a.splits; s += 256) top = __builtin_fmaxf(top, a.part_m[(uint64_t)s * a.n_q + q]);
#pragma unroll
    for (int d = 32; d; d /= 2) top = __builtin_fmaxf(top, __shfl_xor(top, d));
    if (!lane) tops[wave] = top;
    __syncthreads();
    top = __builtin_fmaxf(__builtin_fmaxf(tops[0], tops[1]), __builtin_fmaxf(tops[2], tops[3]));
    const float scale = a.qscale[q], factor = base2(scale), ref = finite_or_zero(top * factor);
    double sum = 0;
    for (uint32_t s = threadIdx.x; s < a.splits; s += 256) {
        const uint64_t at = (uint64_t)s * a.n_q + q;
        sum += (double)a.part_l[at] * (double)__builtin_amdgcn_exp2f(a.part_m[at] * factor - ref);
    }
    sum = wave_sum(sum);
    dot = wave_sum(dot);
    sq = wave_sum(sq);
    if (!lane) {
        sums[wave][0] = sum;
        sums[wave][1] = dot;
        sums[wave][2] = sq;
    }
    __syncthreads();
    if (threadIdx.x) return;
    sum = (sums[0][0] + sums[1][0]) + (sums[2][0] + sums[3][0]);
    dot = (sums[0][1] + sums[1][1]) + (sums[2][1] + sums[3][1]);
    sq = (sums[0][2] + sums[1][2]) + (sums[2][2] + sums[3][2]);
    // The sum is over the reference, a rounded product; taken back to the largest logit itself.
    constexpr double LN2 = 0.693147180559945309417;
    const bool none = top == -__builtin_inff();  // no other candidate
    const double over = none ? -__builtin_inf() : log(sum) - LN2 * __builtin_fmaf(top, factor, -ref);
    const double rest = none ? over : (double)top * scale + over;
    // lse is for the weights, which round every logit to f32: where one has nearly all of the probability it has to be that
    // logit as it is rounded there, and not what a little more than it rounds to.
    const double rest_of_weights = none ? over : (double)(top * scale) + over;
    if (!clicked) {
        loss[q] = 0.0f;
        lse[q] = (float)rest_of_weights;
        return;
    }
    double z = f.scale * dot;
    if (a.norms) {
        const float x = a.norms[click];
        z = x == 0 || sq == 0 ? 0.0 : z / (x * sqrt(sq));
    }
    const double d = rest - z;
    loss[q] = (float)(d > 0 ? d + log1p(exp(-d)) : log1p(exp(d)));
    lse[q] = (float)(d > 0 ? rest_of_weights + log1p(exp(-d)) : z + log1p(exp(d)));
}

// ---- gradients ----------------------------------------------------------------------------

// What the weights of a query with a click have in common.
__device__ __forceinline__ float query_factor(const XentArgs& a, uint32_t q) {
    return (a.grad_loss ? a.grad_loss[q] : 1.0f) * a.qscale[q] * a.sign;
}

// exp(z - lse) of a logit z that has been rounded to f32: where one document has nearly all of the probability, lse is its logit as
// it is rounded here (see join_loss_kernel), and the weight is one (of logits near 100, two that were rounded apart make an error of
// 4e-6). Everything else goes by differences: z log2 e by an fma, and of lse log2 e, whose rounding would be an error of all of
// a query's weights, what is behind it goes into the factor.
struct Base2 {
    float high, rest;
    __device__ __forceinline__ explicit Base2(float lse) {
        high = lse * LOG2E;
        const float low = __builtin_fmaf(lse, LOG2E, -high);
        rest = low == low ? __builtin_amdgcn_exp2f(-low) : 1.0f;
    }
    // over `rest`
    __device__ __forceinline__ static float weight(float z, float high) { return __builtin_amdgcn_exp2f(__builtin_fmaf(z, LOG2E, -high)); }
};

// The weights of the clicked rows of a piece, after weights_kernel, which takes every row alike (to look for them there
// costs two instructions in eight of each element). A clicked row's weight is as large as all others of its query together:
// what its rounding takes away is kept, and goes into the query's gradient at the end.
__global__ __launch_bounds__(256) void click_weights_kernel(XentArgs a) {
    const uint32_t q = blockIdx.x * 256 + threadIdx.x;
    if (q >= a.n_q) return;
    const uint32_t place = a.click[q];
    if (place == NONE || place < a.piece_begin || place - a.piece_begin >= a.piece_rows) return;
    float g = query_factor(a, q) * expm1f(-a.loss[q]);
    if (a.norms) {
        const float x = a.norms[row_at(a, place)];
        g = x == 0 ? 0.0f : g / x;
    }
    char* out = a.g + (uint64_t)(place - a.piece_begin) * a.g_stride + q * 2;
    for (uint32_t p = 0; p < a.g_planes; ++p) {
        const uint32_t bits = bf16_bits(g);
        *reinterpret_cast<uint16_t*>(out + p * a.g_plane) = (uint16_t)bits;
        g -= __builtin_bit_cast(float, bits << 16);
    }
    a.click_rest[q] = g;
}

template <typename S>
using weights_turn = Turn<8, S::UNIT>;

// The weights G of a piece, [candidate][query], kept to 16 bits (PG = 2, of bf16 tables) or all 24 (3) by as many planes of
// bf16. A lane holds four neighbouring queries of a candidate: eight bytes a store. Bound as the loss is, and by what it writes:
// 256 queries over 1M x 768 bf16 570 us (0.69 PFLOP/s; 1 GB written), 256 over 250 thousand x 768 f32 645.
template <typename S, bool NORMS, int PG>
__global__ __launch_bounds__(THREADS, 2) void weights_kernel(XentArgs a) {
    constexpr int BQ = S::Q_TILE;
    extern __shared__ __attribute__((aligned(128))) char lds[];
    __shared__ __attribute__((aligned(16))) float scale[BQ], lse2[BQ], factor[BQ];
    uint32_t tile_q, along;
    place_of_workgroup(a.across, &tile_q, &along);
    const uint32_t q0 = tile_q * BQ;
    const uint32_t end = min(candidates(a), a.piece_begin + a.piece_rows);
    if (end <= a.piece_begin) return;
    if (threadIdx.x < BQ) {
        const uint32_t q = q0 + threadIdx.x;
        const bool in = q < a.n_q && a.click[q] != NONE;
        const Base2 lse(in ? a.lse[q] : 0.0f);
        scale[threadIdx.x] = in ? a.qscale[q] : 0.0f;
        lse2[threadIdx.x] = lse.high;
        factor[threadIdx.x] = in ? query_factor(a, q) * lse.rest : 0.0f;
    }
    // (the first barrier of the loop below orders these before they are read)
    // Every lane stores every time (so that the number of stores is known to the next step's barrier): rows of G are whole
    // tiles of queries, and G is whole tiles of candidates.
    constexpr int UNIT = S::UNIT;
    using T = weights_turn<S>;
    char* const wave_lds = lds + S::LDS + uniform_u32(threadIdx.x >> 6) * T::BYTES;
    S::template run<S::TN * (S::TM / UNIT) * T::STORES * PG>(a, end, q0, along, lds, [&](f32x4 (&acc)[S::TM][S::TN], uint32_t first) {
        const uint32_t l = afresh(threadIdx.x) & 63, row0 = S::wave_r() * S::WR * 16, i0 = S::wave_q() * S::WQ * 16 + (l >> 4) * 4;
        char* out = a.g + (uint64_t)(first - a.piece_begin + row0) * a.g_stride + (q0 + S::wave_q() * S::WQ * 16) * 2;
        float inverse[S::TN];
        if constexpr (NORMS)
#pragma unroll
            for (int n = 0; n < S::TN; ++n) {
                const float x = a.norms[row_at(a, min(first + row0 + (l & 15) + n * 16, end - 1))];
                inverse[n] = x > 0 ? 1.0f / x : 0.0f;
            }
#pragma unroll
        for (int u = 0; u < S::TM / UNIT; ++u)
#pragma unroll
            for (int n = 0; n < S::TN; ++n) {
                Pack<uint16_t, 4> p[UNIT][3];
#pragma unroll
                for (int t = 0; t < UNIT; ++t) {
                    const uint32_t i = i0 + (u * UNIT + t) * 16;
                    const f32x4 vs = *reinterpret_cast<const f32x4*>(scale + i), vl = *reinterpret_cast<const f32x4*>(lse2 + i);
                    const f32x4 vf = *reinterpret_cast<const f32x4*>(factor + i);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        float z = acc[u * UNIT + t][n][r];
                        if constexpr (NORMS) z *= inverse[n];
                        float g = vf[r] * Base2::weight(z * vs[r], vl[r]);
                        if constexpr (NORMS) g *= inverse[n];
                        if constexpr (PG == 2) {
                            // (beyond the largest number of bf16 no number; the general split costs twice the instructions)
                            const uint32_t h = bf16_bits(g);
                            p[t][0].e[r] = (uint16_t)h;
                            p[t][1].e[r] = (uint16_t)bf16_bits(g - __builtin_bit_cast(float, h << 16));
                        } else {
                            const Split x = split(g);
                            p[t][0].e[r] = x.h;
                            p[t][1].e[r] = x.m;
                            p[t][2].e[r] = x.l;
                        }
                    }
                }
#pragma unroll
                for (int k = 0; k < PG; ++k) {
#pragma unroll
                    for (int t = 0; t < UNIT; ++t) T::put(wave_lds, l, t, p[t][k]);
#pragma unroll
                    for (int j = 0; j < T::STORES; ++j)
                        *reinterpret_cast<u32x4*>(out + k * a.g_plane + (uint64_t)(n * 16 + T::row(l, j)) * a.g_stride + u * T::ROW +
                                                  T::chunk(l) * 16) = T::get(wave_lds, l, j);
                }
                __builtin_amdgcn_sched_barrier(0);  // (the registers hold no more at a time)
            }
        return true;
    });
}

// The same of up to four queries, from the products that their loss was made of: a wave takes U neighbouring places at a time.
// Rows of G are those of 64 queries, zeros from NQ on.
template <typename E, typename Q, int V, int NQ, bool NORMS>
__global__ __launch_bounds__(256) void weights_few_kernel(XentArgs a, Few f) {
    using S = FewScores<E, Q, V, NQ, NORMS>;
    constexpr int U = S::U, PG = sizeof(E) == 4 ? 3 : 2;
    extern __shared__ __attribute__((aligned(128))) char lds[];
    __shared__ double sums[4];
    const uint32_t lane = threadIdx.x & 63, wave = uniform_u32(threadIdx.x >> 6), mine = lane % NQ;
    S scores;
    scores.init(a, f, lds, sums);
    const uint32_t end = min(candidates(a), a.piece_begin + a.piece_rows);
    const bool in = a.click[mine] != NONE;
    const Base2 lse(in ? a.lse[mine] : 0.0f);
    const float factor = in ? query_factor(a, mine) * lse.rest : 0.0f;
    for (uint32_t place = a.piece_begin + (blockIdx.x * 4 + wave) * U; place < end; place += gridDim.x * 4 * U) {
        uint32_t row[U];
#pragma unroll
        for (int u = 0; u < U; ++u) row[u] = uniform_u32((uint32_t)row_at(a, min(place + u, end - 1)));
        uint32_t r;
        float length;
        const float z = scores.products(a, f, row, &r, &length);
        float g = factor * Base2::weight(z * scores.scale, lse.high);
        if constexpr (NORMS) g = length == 0 ? 0.0f : g / length;
        const Split x = split(in ? g : 0.0f);
        const uint32_t planes[3] = {x.h, x.m, x.l};
        const uint32_t u = lane / 8, chunk = lane % 8;  // the 16 bytes of a row that the lane stores
#pragma unroll
        for (int k = 0; k < PG; ++k) {
            Pack<uint16_t, 8> p = {};
#pragma unroll
            for (int q = 0; q < NQ; ++q) {
                const uint32_t w = __shfl(planes[k], u * NQ + q);
                p.e[q] = chunk ? 0 : (uint16_t)w;
            }
            if (u < U && place + u < end)
                store_pack<uint16_t, 8>(reinterpret_cast<uint16_t*>(a.g + k * a.g_plane + (uint64_t)(place + u - a.piece_begin) * a.g_stride) + chunk * 8, p);
        }
    }
}

// drows of a piece: transposed queries (BD columns of the rows) by G. The sums are short (for each 64 queries two steps, or six in
// f32) and every one is written: 256 queries, 1M x 768 bf16: 905 us (0.87 PFLOP/s of both planes; 1.5 GB written and 1 read take
// 500 by themselves); 250 thousand x 768 f32: 585 us. A lane holds four neighbouring columns of a row.
// As in weights_kernel every lane stores every time, to its own 16 bytes of a.spill where it has no row or no whole
// 16 bytes of columns; the columns of a last, broken 16 bytes are stored one by one besides.
template <int BD>
constexpr int row_grads_buffers = buffers_of(Rows<BD>::BYTES + Rows<TILE>::BYTES, 8 * 4096);
template <int BD, typename E>
__global__ __launch_bounds__(THREADS, 2) void row_grads_kernel(XentArgs a) {
    using A = Rows<BD>;
    using B = Rows<TILE>;
    constexpr int WAVES_D = 2, WAVES_R = 8 / WAVES_D;
    constexpr int TM = BD / WAVES_D / 16, TN = TILE / WAVES_R / 16;
    extern __shared__ __attribute__((aligned(128))) char lds[];
    const uint32_t wave = uniform_u32(threadIdx.x >> 6), wd = wave % WAVES_D, wr = wave / WAVES_D;
    uint32_t tile_d, along;
    place_of_workgroup(a.across, &tile_d, &along);
    const uint32_t end = min(candidates(a), a.piece_begin + a.piece_rows);
    const uint32_t tiles = end > a.piece_begin ? (end - a.piece_begin + TILE - 1) / TILE : 0;
    if (along >= tiles) return;
    const Planes g{a.g, a.g_plane, a.g_stride, nullptr, end - a.piece_begin, a.gq / 8};
    A q;
    B r;
    q.init();
    r.init();
    q.aim(tile_d * BD);
    r.aim(along * TILE);
    const uint32_t planes = a.grad_steps.n, blocks = a.gq / 64, steps = planes * blocks;
    constexpr int BUFFERS = row_grads_buffers<BD>, BEHIND = (BUFFERS - 2) * (A::LOADS + B::LOADS);
    auto half_q = [&](uint32_t i) { return lds + i * (A::BYTES + B::BYTES); };
    auto half_g = [&](uint32_t i) { return lds + i * (A::BYTES + B::BYTES) + A::BYTES; };
    // (as in Scores::run: the weights are the operand that has further to come)
    Cursor cg{0, 0, along}, cq{0, 0, along};
    auto load_weights = [&](uint32_t to) {
#pragma unroll
        for (int i = 0; i < B::LOADS; ++i) r.load(i, g, cg.k, a.grad_steps.plane_a(cg.c), a.zeros, half_g(to));
        if (cg.advance(planes, blocks, a.splits)) r.aim(cg.tile < tiles ? cg.tile * TILE : NO_ROW);
    };
    auto load_queries = [&](int i, uint32_t to) { q.load(i, a.qt, cq.k, a.grad_steps.plane_b(cq.c), a.zeros, half_q(to)); };
    auto load_all_queries = [&](uint32_t to) {
#pragma unroll
        for (int i = 0; i < A::LOADS; ++i) load_queries(i, to);
        cq.advance(planes, blocks, a.splits);
    };
#pragma unroll
    for (int i = 0; i < BUFFERS - 1; ++i) {
        load_weights(i);
        load_all_queries(i);
    }
    step_barrier<BEHIND>();
    using En = Engine<A, B, TM, TN>;
    En e;
    e.m0 = wd * TM;
    e.n0 = wr * TN;
    e.ask(half_q(0), half_g(0), 0);
    load_weights(BUFFERS - 1);
    uint32_t at = 0;
    constexpr int UNIT = sizeof(E) == 2 ? TM : 4;  // fragments that go through LDS at a time: 256 bytes of a row at most
    using T = Turn<4 * sizeof(E), UNIT>;
    char* const wave_lds = lds + BUFFERS * (A::BYTES + B::BYTES) + wave * T::BYTES;
    uint32_t early = 0, stored = 0;  // as in Scores::run
#pragma nounroll
    for (uint32_t tile = along; tile < tiles; tile += a.splits) {
        f32x4 acc[TM][TN] = {};
#pragma nounroll
        for (uint32_t s = 0; s < steps; ++s) {
            const uint32_t next = at + 1 == BUFFERS ? 0 : at + 1, last = at ? at - 1 : BUFFERS - 1;
            e.template step<BEHIND, TN * (TM / UNIT) * T::STORES>(half_q(at), half_g(at), half_q(next), half_g(next), acc, stored, [&](int phase) {
                if (phase < En::PHASES - 1) {
                    constexpr int EACH = (A::LOADS + En::PHASES - 2) / (En::PHASES - 1);
                    if (BUFFERS == 2 && early) return;
#pragma unroll
                    for (int i = phase * EACH; i < min((phase + 1) * EACH, A::LOADS); ++i) load_queries(i, last);
                    return;
                }
                if (!(BUFFERS == 2 && early)) cq.advance(planes, blocks, a.splits);
                load_weights(at);
                if (BUFFERS > 2) return;
                early = afresh_uniform(s + 1 == steps);
                if (early) load_all_queries(at);
            });
            stored = afresh_uniform(0);
            at = next;
        }
        const uint32_t l = afresh(threadIdx.x) & 63, d0 = tile_d * BD + wd * TM * 16, place0 = a.piece_begin + tile * TILE + wr * TN * 16;
        constexpr uint32_t V = 16 / sizeof(E);
        char* const spill = a.spill + (blockIdx.x * THREADS + threadIdx.x) * 16ull;
        const bool broken = a.dim % V;
#pragma unroll
        for (int n = 0; n < TN; ++n)
#pragma unroll
            for (int u = 0; u < TM / UNIT; ++u) {
#pragma unroll
                for (int t = 0; t < UNIT; ++t) {
                    Pack<E, 4> p;
#pragma unroll
                    for (int i = 0; i < 4; ++i) p.e[i] = from_f32<E>(acc[u * UNIT + t][n][i]);
                    T::put(wave_lds, l, t, p);
                }
#pragma unroll
                for (int j = 0; j < T::STORES; ++j) {
                    const uint32_t place = place0 + n * 16 + T::row(l, j), d = d0 + u * UNIT * 16 + T::chunk(l) * V;
                    E* const out = static_cast<E*>(a.grad_rows) + row_at(a, min(place, end - 1)) * a.grad_row_stride + d;
                    const u32x4 x = T::get(wave_lds, l, j);
                    *reinterpret_cast<typename Words<sizeof(E)>::four*>(place < end && d + V <= a.dim ? (char*)out : spill) = x;
                    if (broken && place < end && d < a.dim && d + V > a.dim) {
                        const Pack<E, V> e = __builtin_bit_cast(Pack<E, V>, x);
#pragma unroll
                        for (uint32_t i = 0; i < V - 1; ++i)
                            if (d + i < a.dim) out[i] = e.e[i];
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        stored = afresh_uniform(1);
    }
    __builtin_amdgcn_s_waitcnt(0x0F70);
}

// dqueries over one share of a piece's candidates: G by rows, the sum running over the candidates. 256 queries over 1M x
// 768 bf16: 745 us (1.05 PFLOP/s of both planes); 1000 over 100 thousand of 200 thousand x 1536, through the list: 560 us (1.10).
// (Through the list two buffers: its reads are waited for with the loads under way counted in, so that only those that
// the barrier has waited for already may be.)
template <int BQ, int BD, bool LISTED>
constexpr int query_grads_buffers = LISTED ? 2 : buffers_of(Cols<BQ>::BYTES + Cols<BD>::BYTES, 0);
template <int BQ, int BD, bool LISTED>
__global__ __launch_bounds__(THREADS, 2) void query_grads_kernel(XentArgs a) {
    using A = Cols<BQ>;
    using B = Cols<BD, LISTED>;
    constexpr int WAVES_Q = BQ >= 128 ? 2 : 1, WAVES_D = 8 / WAVES_Q;
    constexpr int TM = BQ / WAVES_Q / 16, TN = BD / WAVES_D / 16;
    extern __shared__ __attribute__((aligned(128))) char lds[];
    const uint32_t lane = threadIdx.x & 63, wave = uniform_u32(threadIdx.x >> 6), wq = wave % WAVES_Q, wd = wave / WAVES_Q;
    const uint32_t d_tiles = (a.dim + BD - 1) / BD;
    uint32_t tile, share;
    place_of_workgroup(a.across, &tile, &share);
    const uint32_t tile_d = tile % d_tiles, tile_q = tile / d_tiles;
    const uint32_t end = min(candidates(a), a.piece_begin + a.piece_rows);
    const uint32_t n = end > a.piece_begin ? end - a.piece_begin : 0;
    // shares are whole steps of the rows that there are
    const uint32_t per = ((n + STEP - 1) / STEP + a.splits - 1) / a.splits * STEP;
    const uint32_t begin = (uint32_t)min((uint64_t)share * per, (uint64_t)n), stop = min(begin + per, n);
    f32x4 acc[TM][TN] = {};
    const uint32_t blocks = (stop - begin + STEP - 1) / STEP, steps = blocks * a.grad_steps.n;
    if (steps) {
        const Planes g{a.g, a.g_plane, a.g_stride, nullptr, n, a.gq / 8};
        Planes rows = a.rows;
        rows.rows = end - a.place0;
        const uint32_t base = a.piece_begin - a.place0;
        A w;
        B r;
        w.init();
        r.init();
        constexpr int BUFFERS = query_grads_buffers<BQ, BD, LISTED>, BEHIND = (BUFFERS - 2) * (A::LOADS + B::LOADS);
        auto half_g = [&](uint32_t i) { return lds + i * (A::BYTES + B::BYTES); };
        auto half_r = [&](uint32_t i) { return lds + i * (A::BYTES + B::BYTES) + A::BYTES; };
        Cursor cr{0, 0, 0}, cg{0, 0, 0};
        const uint32_t planes = a.grad_steps.n;
        auto load_rows = [&](uint32_t to) {
            const uint32_t from = begin + cr.k * STEP;
#pragma unroll
            for (int i = 0; i < B::LOADS; ++i)
                r.load(i, rows, base + from, base + stop, tile_d * (BD / 8), a.grad_steps.plane_b(cr.c), a.zeros, half_r(to));
            cr.advance(planes, blocks + BUFFERS, 1);  // (behind the last block: zeros)
            if (!cr.c) r.peek(rows, base + from + STEP, base + stop);  // while this step multiplies
        };
        auto load_weights = [&](int i, uint32_t to) {
            w.load(i, g, begin + cg.k * STEP, stop, tile_q * (BQ / 8), a.grad_steps.plane_a(cg.c), a.zeros, half_g(to));
        };
        r.peek(rows, base + begin, base + stop);
#pragma unroll
        for (int i = 0; i < BUFFERS - 1; ++i) {
            load_rows(i);
#pragma unroll
            for (int j = 0; j < A::LOADS; ++j) load_weights(j, i);
            cg.advance(planes, blocks + BUFFERS, 1);
        }
        step_barrier<BEHIND>();
        using En = Engine<A, B, TM, TN>;
        En e;
        e.m0 = wq * TM;
        e.n0 = wd * TN;
        e.ask(half_g(0), half_r(0), 0);
        load_rows(BUFFERS - 1);
        uint32_t at = 0;
#pragma nounroll
        for (uint32_t s = 0; s < steps; ++s) {
            const uint32_t next = at + 1 == BUFFERS ? 0 : at + 1, last = at ? at - 1 : BUFFERS - 1;
            e.template step<BEHIND, 0>(half_g(at), half_r(at), half_g(next), half_r(next), acc, 0, [&](int phase) {
                if (phase == En::PHASES - 1) {
                    cg.advance(planes, blocks + BUFFERS, 1);
                    return load_rows(at);
                }
                constexpr int EACH = (A::LOADS + En::PHASES - 2) / (En::PHASES - 1);
#pragma unroll
                for (int i = phase * EACH; i < min((phase + 1) * EACH, A::LOADS); ++i) load_weights(i, last);
            });
            at = next;
        }
        __builtin_amdgcn_s_waitcnt(0x0F70);
    }
#pragma unroll
    for (int m = 0; m < TM; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t q = tile_q * BQ + (wq * TM + m) * 16 + (lane >> 4) * 4 + i;
            if (q >= a.n_q) continue;
#pragma unroll
            for (int t = 0; t < TN; ++t) {
                const uint32_t d = tile_d * BD + (wd * TN + t) * 16 + (lane & 15);
                if (d >= a.dim) continue;
                float* p = a.part_q + ((uint64_t)share * a.n_q + q) * a.dim + d;
                *p = a.first_piece ? acc[m][t][i] : *p + acc[m][t][i];
            }
        }
}

// The same of an f32 table: G's planes by the rows as they are, split as in SplitScores. 128 queries a tile (256 over 250
// thousand x 768: 570 us, 1.03 PFLOP/s of bf16; by 64 a tile a third more), the LDS of two steps.
constexpr int FLOAT_BD = 128;
template <int BQ, bool LISTED>
constexpr int float_grads_row_buffers = LISTED || BQ > 64 ? 2 : 3;
template <int BQ, bool LISTED>
__global__ __launch_bounds__(THREADS, 2) void float_query_grads_kernel(XentArgs a) {
    using A = Cols<BQ>;
    using B = FloatCols<FLOAT_BD, LISTED>;
    constexpr int WAVES_Q = 2, WAVES_D = 8 / WAVES_Q;
    constexpr int TM = BQ / WAVES_Q / 16, TN = FLOAT_BD / WAVES_D / 16;
    constexpr int ROW_BUFFERS = float_grads_row_buffers<BQ, LISTED>;
    extern __shared__ __attribute__((aligned(128))) char lds[];
    const uint32_t lane = threadIdx.x & 63, wave = uniform_u32(threadIdx.x >> 6), wq = wave % WAVES_Q, wd = wave / WAVES_Q;
    const uint32_t d_tiles = (a.dim + FLOAT_BD - 1) / FLOAT_BD;
    uint32_t tile, share;
    place_of_workgroup(a.across, &tile, &share);
    const uint32_t tile_d = tile % d_tiles, tile_q = tile / d_tiles;
    const uint32_t end = min(candidates(a), a.piece_begin + a.piece_rows);
    const uint32_t n = end > a.piece_begin ? end - a.piece_begin : 0;
    const uint32_t per = ((n + STEP - 1) / STEP + a.splits - 1) / a.splits * STEP;
    const uint32_t begin = (uint32_t)min((uint64_t)share * per, (uint64_t)n), stop = min(begin + per, n);
    f32x4 acc[TM][TN] = {}, small[TM][TN] = {};
    const uint32_t steps = (stop - begin + STEP - 1) / STEP;
    if (steps) {
        const Planes g{a.g, a.g_plane, a.g_stride, nullptr, n, a.gq / 8};
        Planes rows = a.rows;
        rows.rows = end - a.place0;
        const uint32_t base = a.piece_begin - a.place0;
        A w;
        B r;
        w.init();
        r.init();
        auto half_r = [&](uint32_t i) { return lds + i * B::BYTES; };
        auto half_g = [&](uint32_t i) { return lds + ROW_BUFFERS * B::BYTES + i * 3 * A::BYTES; };
        uint32_t kr = begin, kg = begin;
        auto load_rows = [&](uint32_t to) {
#pragma unroll
            for (int i = 0; i < B::LOADS; ++i) r.load(i, rows, base + kr, base + stop, tile_d * (FLOAT_BD / 4), a.zeros, half_r(to));
            kr += STEP;
            r.peek(rows, base + kr, base + stop);  // while this step multiplies
        };
        auto load_weights = [&](uint32_t to) {
#pragma unroll
            for (int p = 0; p < 3; ++p)
#pragma unroll
                for (int i = 0; i < A::LOADS; ++i) w.load(i, g, kg, stop, tile_q * (BQ / 8), p, a.zeros, half_g(to) + p * A::BYTES);
            kg += STEP;
        };
        constexpr int BEHIND = (ROW_BUFFERS - 2) * B::LOADS;
        r.peek(rows, base + begin, base + stop);
        load_weights(0);
        load_rows(0);
        load_weights(1);
        load_rows(1);
        step_barrier<3 * A::LOADS + B::LOADS>();
        SplitEngine<A, B, TM, TN, true> e;
        e.p0 = wq * TM;
        e.x0 = wd * TN;
        e.start(half_g(0), half_r(0));
        if (ROW_BUFFERS > 2) load_rows(2);
        uint32_t at_r = 0, at_g = 0;
#pragma nounroll
        for (uint32_t s = 0; s < steps; ++s) {
            const uint32_t next_r = at_r + 1 == ROW_BUFFERS ? 0 : at_r + 1, next_g = at_g ^ 1;
            e.template half<0>([] {}, half_g(at_g), half_r(at_r), 1, acc, small, [] {});
            e.template half<1>([] { step_barrier<BEHIND>(); }, half_g(next_g), half_r(next_r), 0, acc, small, [&] {
                load_weights(at_g);
                load_rows(at_r);
            });
            at_r = next_r;
            at_g = next_g;
        }
        __builtin_amdgcn_s_waitcnt(0x0F70);
    }
#pragma unroll
    for (int m = 0; m < TM; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t q = tile_q * BQ + (wq * TM + m) * 16 + (lane >> 4) * 4 + i;
            if (q >= a.n_q) continue;
#pragma unroll
            for (int t = 0; t < TN; ++t) {
                const uint32_t d = tile_d * FLOAT_BD + (wd * TN + t) * 16 + (lane & 15);
                if (d >= a.dim) continue;
                float* p = a.part_q + ((uint64_t)share * a.n_q + q) * a.dim + d;
                const float sum = acc[m][t][i] + small[m][t][i];
                *p = a.first_piece ? sum : *p + sum;
            }
        }
}

// The shares of a query's gradient joined, and taken through the query's length where logits are cosines; one
// workgroup per (query, 256 columns), or per query where its length is needed.
template <typename E, typename Q, typename O>
__global__ __launch_bounds__(256) void join_query_grads_kernel(XentArgs a, Few f, O* out, uint64_t out_stride) {
    __shared__ double sums[8];
    const uint32_t q = blockIdx.x;
    if (a.click[q] == NONE) {
        for (uint32_t d = blockIdx.y * 256 + threadIdx.x; d < a.dim; d += gridDim.y * 256) out[q * out_stride + d] = from_f32<O>(0.0f);
        return;
    }
    const Q* const query = static_cast<const Q*>(f.queries) + q * f.query_stride;
    const E* const clicked = static_cast<const E*>(f.rows) + (f.targets[q] - f.first_id) * f.stride;
    const float rest = a.click_rest[q];
    float* sum0 = a.part_q + (uint64_t)q * a.dim;
    double dot = 0, sq = 0;  // (as in pack_queries_kernel)
    for (uint32_t d = blockIdx.y * 256 + threadIdx.x; d < a.dim; d += gridDim.y * 256) {
        // (64 bits: the clicked row's share is as large as all others together, which would be added to it last bit by last bit)
        double all = sizeof(E) == 2 ? rest * to_f32(clicked[d]) : 0.0f;  // (of three planes nothing is left)
#pragma unroll 8
        for (uint32_t s = 0; s < a.splits; ++s) all += a.part_q[((uint64_t)s * a.n_q + q) * a.dim + d];
        const float sum = (float)all;
        if (!a.norms) {
            out[q * out_stride + d] = from_f32<O>(sum);
            continue;
        }
        const double x = query_element<E>(query[d]);
        dot += sum * x;
        sq += x * x;
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
    const double along = sq > 0 ? dot / sq : 0.0;
    for (uint32_t d = threadIdx.x; d < a.dim; d += 256) {
        const double x = query_element<E>(query[d]);
        out[q * out_stride + d] = from_f32<O>((float)(sum0[d] - along * x));
    }
}

// Rows that are no candidates have gradient zero (`all`: every row, where there is no query). A wave a row: 7 us for a tenth
// of 50 thousand.
template <typename E>
__global__ __launch_bounds__(256) void clear_rows_kernel(const uint64_t* mask, const uint64_t* present, bool all, uint64_t n_rows,
                                                         uint32_t dim, E* out, uint64_t stride) {
    for (uint64_t r = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < n_rows; r += (uint64_t)gridDim.x * 4) {
        if (!all && word_at(mask, present, r >> 6, n_rows) >> (r & 63) & 1) continue;
        for (uint32_t d = threadIdx.x & 63; d < dim; d += 64) out[r * stride + d] = from_f32<E>(0.0f);
    }
}

// ---- host side ----------------------------------------------------------------------------

constexpr uint64_t PIECE_BYTES = 1u << 30;  // of weights, and of planes, that are held at a time (a quarter of it, a piece that the
                                            // memory-side cache holds, costs more in launches than it saves)
constexpr uint32_t WORKGROUPS = 256;          // of a product: one per CU (the LDS of a tile fills one)
constexpr uint32_t FEW_WORKGROUPS = 2048;     // of the loss of a few queries: eight per CU

// hh, hm, mh, mm, hl, lh | planes 0 and 1 of A
constexpr Steps SIX{6, 0u | 0u << 2 | 1u << 4 | 1u << 6 | 0u << 8 | 2u << 10, 0u | 1u << 2 | 0u << 4 | 1u << 6 | 2u << 8 | 0u << 10};
constexpr Steps TWO{2, 0u | 1u << 2, 0};

// Up to four queries by plain products, which need no list of candidates and no planes of queries: rows of f32 always (200
// thousand x 768, four queries: 115 us, on the matrix cores 164), rows of bf16 while their bytes still bound them (one
// query over 1M x 768: 238 us and 260; two 260 and 261, three 276 and 260, four 320 and 261) or launches do (20 thousand x
// 384, a fifth of them: four queries 16 us and 26). Queries of all lanes' columns have to fit LDS.
bool few_queries(uint32_t n_q, uint64_t n_rows, uint32_t dim, int32_t dtype) {
    const bool bound = dtype == VS_F32 || n_rows * dim * 2 <= 256u << 20;
    return n_q <= (bound ? 4 : 2) && n_q * (uint64_t)dim <= 12288;
}

struct Plan {
    bool few;
    uint32_t planes, g_planes, kp, gq, score_bq, score_rows, bq, bd, q_tiles, score_q_tiles, d_tiles, grad_d_tiles;
    uint32_t score_splits, row_splits, grad_splits;
    uint64_t piece_rows, packed_rows;
};

// Workgroups along the rows for `across` side by side: one round of the CUs (a workgroup more would take a second one).
uint32_t splits_for(uint32_t across, uint64_t tiles) {
    return (uint32_t)std::min<uint64_t>(std::max<uint64_t>(WORKGROUPS / across, 1), tiles);
}

Plan plan_for(uint32_t n_q, uint64_t n_rows, uint32_t dim, int32_t dtype) {
    Plan p;
    p.few = few_queries(n_q, n_rows, dim, dtype);
    p.planes = dtype == VS_F32 ? 3 : 1;
    // Weights of a bf16 table have 16 bits. Rounded to bf16, 2^-8 of each at most, they would be as far off as a gradient's own
    // rounding is, and further where a gradient is the difference of terms that nearly cancel, as those of a clicked document and
    // a copy of it do. (The price: loss and gradients of 256 queries over 1M x 768 take 2.65 ms, 1.93 with bf16 weights; of 1000
    // over half of 200 thousand x 1536, queries' alone, 1.24 and 0.94.)
    p.g_planes = dtype == VS_F32 ? 3 : 2;
    p.kp = (uint32_t)round_up(dim, 64);
    p.gq = (uint32_t)round_up(n_q, 64);
    p.bq = n_q <= 64 ? 64 : n_q <= 128 || dtype == VS_F32 ? 128 : 256;
    p.score_bq = dtype == VS_F32 ? 64 : p.bq;
    // an odd number of 128 columns by 128 at a time: no half-empty tiles (200 thousand x 384, 128 queries: rows' gradients
    // 82 us, 89 by 256; queries' 61 and 65)
    p.bd = (dim + 127) / 128 % 2 ? 128 : 256;
    p.score_q_tiles = (n_q + p.score_bq - 1) / p.score_bq;
    p.q_tiles = (n_q + p.bq - 1) / p.bq;
    p.d_tiles = (dim + p.bd - 1) / p.bd;
    p.grad_d_tiles = dtype == VS_F32 ? (dim + FLOAT_BD - 1) / FLOAT_BD : p.d_tiles;
    const uint64_t rows = round_up(n_rows, TILE), per = TILE * (uint64_t)WORKGROUPS;
    auto piece = [&](uint64_t row_bytes) {
        uint64_t r = std::max<uint64_t>(PIECE_BYTES / row_bytes / TILE * TILE, TILE);
        if (r > per) r = r / per * per;  // whole rounds of the workgroups
        return std::min(r, rows);
    };
    p.piece_rows = piece((uint64_t)p.q_tiles * p.bq * 2 * p.g_planes);
    p.packed_rows = std::min(p.piece_rows, piece((uint64_t)p.kp * (dtype == VS_F32 ? 4 : 2)));
    const uint64_t tiles = rows / TILE;
    // f32 rows by 256 a tile, or by 128 where that leaves CUs idle for most of a round (256 queries, 250 thousand rows: 664 us
    // and 813; 100 queries, 50 thousand: 52 and 43), or by 64 where all tiles have a CU then (64 queries, 10 thousand x 384:
    // 13 us and 17 by 128; 30, 20 thousand x 768, which take two rounds: 35 and 28)
    const uint64_t score_tiles_256 = p.score_q_tiles * tiles;
    p.score_rows = dtype != VS_F32 || score_tiles_256 >= 2 * WORKGROUPS ? TILE : score_tiles_256 * 4 > WORKGROUPS ? 128 : 64;
    const uint64_t score_tiles = rows / p.score_rows;
    p.score_splits = splits_for(p.score_q_tiles, score_tiles);
    p.row_splits = splits_for(p.d_tiles, tiles);
    p.grad_splits = splits_for(p.q_tiles * p.grad_d_tiles, tiles * (TILE / STEP));
    return p;
}

// Workgroups of the list of candidates. Up to LIST_ALONE of them each counts the words before its own: a launch less (31
// of them, 500 thousand rows: 13.7 us so, 9.5 with counts made first; 977, 16 million rows: 395 and 19).
uint32_t list_blocks(uint64_t n_rows) { return (uint32_t)(((n_rows + 63) / 64 + LIST_WORDS - 1) / LIST_WORDS); }
constexpr uint32_t LIST_ALONE = 8;

struct Buffers {
    uint32_t *zeros, *list, *count, *sums, *click;
    float *qscale, *click_rest, *part_m, *part_l, *part_q;
    char *q, *qt, *g, *packed, *spill;
    uint64_t bytes;
};
// What a call does not use is not there: of the loss of few queries all but its shares, of other losses what belongs to the
// gradients, of rows that are aligned their copies.
Buffers carve(void* workspace, const Plan& p, uint32_t n_q, uint64_t n_rows, uint32_t dim, bool aligned, bool gradients) {
    Carver w(workspace);
    Buffers b{};
    if (!gradients) {
        const uint64_t parts = n_q * (uint64_t)(p.few ? FEW_WORKGROUPS : p.score_splits);
        b.part_m = w.take<float>(parts);
        b.part_l = w.take<float>(parts);
        if (p.few) {
            b.qscale = w.take<float>(n_q);
            b.bytes = w.at() - (char*)workspace;
            return b;
        }
    }
    b.zeros = w.take<uint32_t>(64);
    b.list = w.take<uint32_t>(n_rows);
    b.count = w.take<uint32_t>(1);
    b.sums = w.take<uint32_t>(list_blocks(n_rows));
    b.click = w.take<uint32_t>(n_q);
    b.qscale = w.take<float>(n_q);
    b.q = w.take<char>((uint64_t)n_q * p.kp * 2 * p.planes);
    if (gradients) {
        b.click_rest = w.take<float>(n_q);
        b.qt = w.take<char>((uint64_t)dim * p.gq * 2 * p.planes);
        b.g = w.take<char>(p.piece_rows * p.q_tiles * p.bq * 2 * p.g_planes);
        b.spill = w.take<char>(16ull * THREADS * WORKGROUPS);
        b.part_q = w.take<float>((uint64_t)p.grad_splits * n_q * dim);
    }
    if (!aligned) b.packed = w.take<char>(p.packed_rows * p.kp * (p.planes == 3 ? 4 : 2));
    b.bytes = w.at() - (char*)workspace;
    return b;
}

Few few_of(const Xent& x) {
    return Few{x.t.rows, x.queries, x.t.stride, x.query_stride, x.targets, x.mask, x.t.present, x.t.first_id, x.scale, 1};
}

// A call's plan, buffers and arguments.
struct Call {
    const Xent& x;
    Plan p;
    Buffers b;
    XentArgs a{};
    bool packed;
    hipStream_t stream;
    hipError_t error = hipSuccess;

    Call(const Xent& x_, void* workspace, bool gradients, hipStream_t stream_)
        : x(x_), p(plan_for(x.n_q, x.t.n_rows, x.t.dim, x.t.dtype)),
          b(carve(workspace, p, x.n_q, x.t.n_rows, x.t.dim, rows_are_aligned(x.t), gradients)), stream(stream_) {
        const uint32_t dim = x.t.dim;
        const uint32_t size = x.t.dtype == VS_F32 ? 4 : 2, chunk = 16 / size;
        packed = !rows_are_aligned(x.t);
        a.n_rows = x.t.n_rows;
        a.norms = x.norms;
        a.q = Planes{b.q, (uint64_t)x.n_q * p.kp * 2, p.kp * 2, nullptr, x.n_q, p.kp / 8};
        a.qt = Planes{b.qt, (uint64_t)dim * p.gq * 2, p.gq * 2, nullptr, dim, p.gq / 8};
        a.n_q = x.n_q;
        a.gq = p.gq;
        a.dim = dim;
        a.click = b.click;
        a.qscale = b.qscale;
        a.sign = x.scale < 0 ? -1.0f : 1.0f;
        a.grad_steps = p.planes == 3 ? SIX : TWO;
        a.zeros = (const char*)b.zeros;
        a.part_m = b.part_m;
        a.part_l = b.part_l;
        a.g = b.g;
        a.g_stride = p.q_tiles * p.bq * 2;
        a.g_planes = p.g_planes;
        a.click_rest = b.click_rest;
        a.g_plane = p.piece_rows * a.g_stride;
        a.spill = b.spill;
        a.part_q = b.part_q;
        if (x.mask || x.t.present) {
            a.list = b.list;
            a.count = b.count;
            const uint32_t blocks = list_blocks(x.t.n_rows), *sums = blocks > LIST_ALONE ? b.sums : nullptr;
            if (sums) count_words_kernel<<<blocks, 256, 0, stream>>>(x.mask, x.t.present, x.t.n_rows, b.sums);
            list_candidates_kernel<<<blocks, 256, 0, stream>>>(x.mask, x.t.present, x.t.n_rows, sums, b.list, b.count);
        }
        a.rows = packed ? Planes{b.packed, 0, p.kp * size, nullptr, 0, p.kp / chunk}
                        : Planes{(const char*)x.t.rows, 0, (uint32_t)x.t.stride * size, a.list, 0, dim / chunk};
        const uint32_t grid = p.gq / 64 * (p.kp / 64) + (x.n_q + 3) / 4;
        auto pack = [&](auto kernel) { kernel<<<grid, 256, 0, stream>>>(a, few_of(x), b.click, b.qscale, b.zeros, gradients); };
        if (x.t.dtype == VS_F32)
            pack(pack_queries_kernel<float, 3>);
        else if (x.queries_f32)
            pack(pack_queries_kernel<float, 1>);
        else
            pack(pack_queries_kernel<bf16, 1>);
    }

    // `body` for every piece of the candidates, of at most `rows`, its planes ready.
    template <typename F>
    void for_pieces(uint64_t rows, F&& body) {
        for (uint64_t begin = 0; begin < x.t.n_rows; begin += rows) {
            a.piece_begin = (uint32_t)begin;
            a.piece_rows = (uint32_t)std::min(rows, x.t.n_rows - begin);
            a.first_piece = !begin;
            a.place0 = packed ? a.piece_begin : 0;
            if (packed) pack_rows();
            body();
        }
    }

    void pack_rows() {
        const uint64_t threads = (uint64_t)a.piece_rows * a.rows.chunks;
        const uint32_t grid = (uint32_t)std::min<uint64_t>((threads + 255) / 256, 1u << 16);
        if (x.t.dtype == VS_F32)
            pack_rows_kernel<float><<<grid, 256, 0, stream>>>(a, (const float*)x.t.rows, x.t.stride, b.packed);
        else
            pack_rows_kernel<bf16><<<grid, 256, 0, stream>>>(a, (const bf16*)x.t.rows, x.t.stride, b.packed);
    }

    // A product over the tiles of the piece.
    template <typename K>
    void product(K kernel, uint32_t lds, uint32_t across, uint32_t splits) {
        a.across = across;
        a.splits = splits;
        if (error == hipSuccess) error = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (error == hipSuccess) kernel<<<across * splits, THREADS, lds, stream>>>(a);
    }

    // Calls `f` with a Scores type for tiles of BQ queries and whether logits are cosines, as constants.
    template <int BQ, bool LANES_ARE_QUERIES, typename F>
    void with_scores(F&& f) {
        auto by_norms = [&](auto scores) { a.norms ? f(scores, std::true_type{}) : f(scores, std::false_type{}); };
        if constexpr (BQ == 64)
            if (p.planes == 3) {
                auto by_list = [&](auto rows) {
                    if (a.rows.list) return by_norms(SplitScores<LANES_ARE_QUERIES, true, rows>{});
                    by_norms(SplitScores<LANES_ARE_QUERIES, false, rows>{});
                };
                if (p.score_rows == 256) return by_list(std::integral_constant<int, 256>{});
                if (p.score_rows == 128) return by_list(std::integral_constant<int, 128>{});
                return by_list(std::integral_constant<int, 64>{});
            }
        if (a.rows.list) return by_norms(Scores<BQ, LANES_ARE_QUERIES, true>{});
        by_norms(Scores<BQ, LANES_ARE_QUERIES, false>{});
    }

    template <int BQ>
    void loss() {
        with_scores<BQ, true>([&](auto scores, auto norms) {
            using S = decltype(scores);
            product(loss_kernel<S, norms>, S::LDS, p.score_q_tiles, p.score_splits);
        });
    }

    template <int BQ, int PG>
    void weights() {
        with_scores<BQ, false>([&](auto scores, auto norms) {
            using S = decltype(scores);
            // (three planes of weights are an f32 table's)
            if constexpr ((PG == 3) == S::SPLIT)
                product(weights_kernel<S, norms, PG>, S::LDS + 8 * weights_turn<S>::BYTES, p.score_q_tiles, p.score_splits);
        });
    }
    template <int BQ>
    void weights() {
        if constexpr (BQ == 64)
            p.planes == 3 ? weights<BQ, 3>() : weights<BQ, 2>();
        else
            weights<BQ, 2>();
    }

    template <int BD, typename E>
    void row_grads() {
        // (and a Turn's rows for every wave)
        product(row_grads_kernel<BD, E>, row_grads_buffers<BD> * (Rows<BD>::BYTES + Rows<TILE>::BYTES) + 8 * 4096, p.d_tiles, p.row_splits);
    }
    template <typename E>
    void row_grads() {
        p.bd == 256 ? row_grads<256, E>() : row_grads<128, E>();
    }

    template <int BQ, int BD, bool LISTED>
    void query_grads() {
        product(query_grads_kernel<BQ, BD, LISTED>, query_grads_buffers<BQ, BD, LISTED> * (Cols<BQ>::BYTES + Cols<BD>::BYTES),
                p.q_tiles * p.d_tiles, p.grad_splits);
    }
    template <int BQ>
    void query_grads() {
        if (a.rows.list)
            p.bd == 256 ? query_grads<BQ, 256, true>() : query_grads<BQ, 128, true>();
        else
            p.bd == 256 ? query_grads<BQ, 256, false>() : query_grads<BQ, 128, false>();
    }
    template <int BQ>
    void float_query_grads() {
        auto run = [&](auto kernel, int row_buffers) {
            product(kernel, 2 * 3 * Cols<BQ>::BYTES + row_buffers * FloatCols<FLOAT_BD>::BYTES, p.q_tiles * p.grad_d_tiles, p.grad_splits);
        };
        if (a.rows.list)
            run(float_query_grads_kernel<BQ, true>, float_grads_row_buffers<BQ, true>);
        else
            run(float_query_grads_kernel<BQ, false>, float_grads_row_buffers<BQ, false>);
    }

    template <typename E, typename Q, typename O>
    void join_query_grads(void* out, uint64_t out_stride) {
        a.splits = p.grad_splits;
        const dim3 grid(x.n_q, a.norms ? 1 : (a.dim + 255) / 256);
        join_query_grads_kernel<E, Q, O><<<grid, 256, 0, stream>>>(a, few_of(x), (O*)out, out_stride);
    }
};

// Calls `f` with FewScores for a few queries of this call, as a type.
template <typename E, typename Q, int V, typename F>
void with_few_scores(uint32_t n_q, bool norms, F&& f) {
    auto by_norms = [&](auto nq) {
        if (norms)
            f(FewScores<E, Q, V, nq, true>{}, nq, std::true_type{});
        else
            f(FewScores<E, Q, V, nq, false>{}, nq, std::false_type{});
    };
    switch (n_q) {
        case 1: return by_norms(std::integral_constant<int, 1>{});
        case 2: return by_norms(std::integral_constant<int, 2>{});
        case 3: return by_norms(std::integral_constant<int, 3>{});
        default: return by_norms(std::integral_constant<int, 4>{});
    }
}
uint32_t few_lds(uint32_t n_q, uint32_t dim, uint32_t v) { return n_q * (uint32_t)round_up(dim, v) * 4; }

template <typename E, typename Q, int V>
hipError_t run_loss_few(const Xent& x, XentArgs a, const Few& f, float* qscale, float* loss, float* lse, hipStream_t stream) {
    a.splits = (uint32_t)std::min<uint64_t>(((x.t.n_rows + 63) / 64 * f.parts + 3) / 4, FEW_WORKGROUPS);
    with_few_scores<E, Q, V>(x.n_q, a.norms, [&](auto, auto nq, auto norms) {
        loss_few_kernel<E, Q, V, nq, norms><<<a.splits, 256, few_lds(x.n_q, a.dim, V), stream>>>(a, f, qscale);
    });
    a.qscale = qscale;
    join_loss_kernel<E, Q><<<x.n_q, 256, 0, stream>>>(a, f, loss, lse);
    return hipGetLastError();
}
hipError_t launch_loss_few(const Xent& x, void* workspace, float* loss, float* lse, hipStream_t stream) {
    const Buffers b = carve(workspace, plan_for(x.n_q, x.t.n_rows, x.t.dim, x.t.dtype), x.n_q, x.t.n_rows, x.t.dim, true, false);
    XentArgs a{};
    a.n_rows = x.t.n_rows;
    a.dim = x.t.dim;
    a.n_q = x.n_q;
    a.norms = x.norms;
    a.part_m = b.part_m;
    a.part_l = b.part_l;
    Few f = few_of(x);
    // small tables: parts of a word, down to eight rows, until there is one for every wave
    while (f.parts < 8 && (x.t.n_rows + 63) / 64 * f.parts * 2 <= FEW_WORKGROUPS * 4) f.parts *= 2;
    if (x.t.dtype == VS_F32) return run_loss_few<float, float, 4>(x, a, f, b.qscale, loss, lse, stream);
    return x.queries_f32 ? run_loss_few<bf16, float, 8>(x, a, f, b.qscale, loss, lse, stream) : run_loss_few<bf16, bf16, 8>(x, a, f, b.qscale, loss, lse, stream);
}

template <typename E, typename Q, int V>
void run_weights_few(const Xent& x, const XentArgs& a, hipStream_t stream) {
    with_few_scores<E, Q, V>(x.n_q, a.norms, [&](auto scores, auto nq, auto norms) {
        constexpr uint32_t each = 4 * decltype(scores)::U;
        weights_few_kernel<E, Q, V, nq, norms>
            <<<std::min((a.piece_rows + each - 1) / each, FEW_WORKGROUPS), 256, few_lds(x.n_q, a.dim, V), stream>>>(a, few_of(x));
    });
}
void weights_few(const Xent& x, const XentArgs& a, hipStream_t stream) {
    if (x.t.dtype == VS_F32)
        run_weights_few<float, float, 4>(x, a, stream);
    else if (x.queries_f32)
        run_weights_few<bf16, float, 8>(x, a, stream);
    else
        run_weights_few<bf16, bf16, 8>(x, a, stream);
}

void clear_rows(const Xent& x, void* grad_rows, uint64_t stride, bool all, hipStream_t stream) {
    const uint32_t grid = (uint32_t)std::min<uint64_t>((x.t.n_rows + 3) / 4, 1u << 16);
    if (x.t.dtype == VS_F32)
        clear_rows_kernel<<<grid, 256, 0, stream>>>(x.mask, x.t.present, all, x.t.n_rows, x.t.dim, (float*)grad_rows, stride);
    else
        clear_rows_kernel<<<grid, 256, 0, stream>>>(x.mask, x.t.present, all, x.t.n_rows, x.t.dim, (bf16*)grad_rows, stride);
}

}  // namespace

bool rows_are_aligned(const Table& t) {
    const uint32_t size = t.dtype == VS_F32 ? 4 : 2, chunk = 16 / size;
    return (uintptr_t)t.rows % 16 == 0 && t.stride % chunk == 0 && t.stride * size <= 0xFFFFFFFFu && t.dim % chunk == 0;
}

uint64_t xent_workspace_bytes(uint32_t n_q, uint64_t n_rows, uint32_t dim, int32_t dtype, bool aligned, bool gradients) {
    return carve(nullptr, plan_for(n_q, n_rows, dim, dtype), n_q, n_rows, dim, aligned, gradients).bytes + 256;
}

hipError_t launch_xent(const Xent& x, void* workspace, float* loss, float* lse, hipStream_t stream) {
    if (few_queries(x.n_q, x.t.n_rows, x.t.dim, x.t.dtype)) return launch_loss_few(x, workspace, loss, lse, stream);
    Call c(x, workspace, false, stream);
    c.for_pieces(c.packed ? c.p.packed_rows : x.t.n_rows, [&] {
        c.p.score_bq == 64 ? c.loss<64>() : c.p.score_bq == 128 ? c.loss<128>() : c.loss<256>();
    });
    c.a.splits = c.p.score_splits;
    if (c.error != hipSuccess) return c.error;
    auto join = [&](auto kernel) { kernel<<<x.n_q, 256, 0, stream>>>(c.a, few_of(x), loss, lse); };
    if (x.t.dtype == VS_F32)
        join(join_loss_kernel<float, float>);
    else if (x.queries_f32)
        join(join_loss_kernel<bf16, float>);
    else
        join(join_loss_kernel<bf16, bf16>);
    return hipGetLastError();
}

hipError_t launch_xent_grad(const Xent& x, const float* loss, const float* lse, const float* grad_loss, void* workspace,
                            void* grad_queries, uint64_t grad_query_stride, void* grad_rows, uint64_t grad_row_stride,
                            hipStream_t stream) {
    if (!x.n_q) {
        if (grad_rows) clear_rows(x, grad_rows, grad_row_stride, true, stream);
        return hipGetLastError();
    }
    if (!grad_queries && !grad_rows) return hipSuccess;
    Call c(x, workspace, true, stream);
    c.a.loss = loss;
    c.a.lse = lse;
    c.a.grad_loss = grad_loss;
    c.a.grad_rows = grad_rows;
    c.a.grad_row_stride = grad_row_stride;
    const bool f32 = x.t.dtype == VS_F32;
    if (grad_rows && c.a.list) clear_rows(x, grad_rows, grad_row_stride, false, stream);
    c.for_pieces(c.packed ? c.p.packed_rows : c.p.piece_rows, [&] {
        if (c.p.few)
            weights_few(x, c.a, stream);
        else
            c.p.score_bq == 64 ? c.weights<64>() : c.p.score_bq == 128 ? c.weights<128>() : c.weights<256>();
        if (c.error == hipSuccess) click_weights_kernel<<<(x.n_q + 255) / 256, 256, 0, stream>>>(c.a);
        if (grad_rows) f32 ? c.row_grads<float>() : c.row_grads<bf16>();
        if (!grad_queries) return;
        if (f32) return c.p.bq == 64 ? c.float_query_grads<64>() : c.float_query_grads<128>();
        c.p.bq == 64 ? c.query_grads<64>() : c.p.bq == 128 ? c.query_grads<128>() : c.query_grads<256>();
    });
    if (c.error != hipSuccess) return c.error;
    if (grad_queries) {
        if (f32)
            c.join_query_grads<float, float, float>(grad_queries, grad_query_stride);
        else if (x.queries_f32)
            c.join_query_grads<bf16, float, float>(grad_queries, grad_query_stride);
        else
            c.join_query_grads<bf16, bf16, bf16>(grad_queries, grad_query_stride);
    }
    return hipGetLastError();
}

}  // namespace learn
}  // namespace vs
