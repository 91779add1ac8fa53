// Pooled row lookup and its gradients.
//
//   out[b]  = scale * sum over i in bag b of w[i] * rows[ids[i]]
//   drows[r] = scale * sum over i with ids[i] = r of w[i] * g[bag(i)]
//   dw[i]   = scale * <rows[ids[i]], g[bag(i)]>
//
// All of it is bound by memory: two operations per element read. Sums are f32 in a fixed order (no
// atomics), rounded once when they are stored; a call gives the same bits every time.
#include "../../include/vs_abi.h"
#include "learn_kernels.h"
#include "learn_device.h"

namespace vs {
namespace learn {
namespace {

constexpr uint32_t NONE = 0xFFFFFFFFu;

struct LookupArgs {
    Table t;
    Bags b;
    void* out;
    uint64_t out_stride;
    uint32_t chunks;  // pieces of V columns in a row
};

// Position p's row, or NONE for an id that names none.
__device__ __forceinline__ uint32_t row_of(const Table& t, uint32_t id) {
    const uint32_t r = id - t.first_id;
    if (id < t.first_id || r >= t.n_rows) return NONE;
    if (t.present && !(t.present[r >> 6] >> (r & 63) & 1)) return NONE;
    return r;
}

__device__ __forceinline__ void bag_range(const Bags& b, uint64_t bag, uint64_t* begin, uint64_t* end) {
    if (!b.offsets) {
        *begin = bag;
        *end = bag < b.n_ids ? bag + 1 : bag;
        return;
    }
    // offsets are device data that nobody has checked: what they name stays inside ids[n_ids]
    const uint64_t lo = b.offsets[bag], hi = b.offsets[bag + 1];
    *end = hi < b.n_ids ? hi : b.n_ids;
    *begin = lo < *end ? lo : *end;
}

// acc += the weighted rows at positions begin, begin + step, .. < end, of a piece of V columns.
// Four rows are in flight at a time; a position without a row adds nothing (its load goes to row 0, and what that
// holds, not even a NaN, gets into the sum).
template <typename E, int V>
__device__ __forceinline__ void add_rows(const LookupArgs& a, uint64_t begin, uint64_t end, uint32_t step,
                                         const Piece<V>& piece, float (&acc)[V]) {
    constexpr int U = 4;
    const E* rows = static_cast<const E*>(a.t.rows);
    for (uint64_t i = begin; i < end; i += (uint64_t)U * step) {
        uint32_t r[U];
        float w[U];
        Pack<E, V> x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint64_t p = i + (uint64_t)u * step;
            const bool in = p < end;
            r[u] = in ? row_of(a.t, a.b.ids[p]) : NONE;
            w[u] = in && a.b.weights ? a.b.weights[p] : 1.0f;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] = load_piece<E, V>(rows + (uint64_t)(r[u] == NONE ? 0 : r[u]) * a.t.stride, piece, a.t.dim);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int v = 0; v < V; ++v) acc[v] = r[u] == NONE ? acc[v] : __builtin_fmaf(w[u], to_f32(x[u].e[v]), acc[v]);
    }
}

template <typename O, int V>
__device__ __forceinline__ void store_out(const LookupArgs& a, uint64_t bag, const Piece<V>& piece, const float (&acc)[V]) {
    Pack<O, V> p;
#pragma unroll
    for (int v = 0; v < V; ++v) p.e[v] = from_f32<O>(acc[v] * a.b.scale);
    store_piece<O, V>(static_cast<O*>(a.out) + bag * a.out_stride, piece, a.t.dim, p, false);
}

// One thread per (bag, V columns): a wave reads 64 neighbouring pieces of a row (1 KiB of 16-byte pieces), and no lane
// idles whatever the row's length. 16384 bags of 0 to 40 of 1M x 768 bf16: 100 us, 5.0 TB/s of rows (popular ones come from
// cache); one bag of three: 3.5 us, two trips to memory.
template <typename E, typename O, int V>
__global__ __launch_bounds__(256) void lookup_kernel(LookupArgs a) {
    const uint64_t total = a.b.n_bags * a.chunks;
    for (uint64_t base = (uint64_t)blockIdx.x * 256; base < total; base += (uint64_t)gridDim.x * 256) {
        if (base + threadIdx.x >= total) break;
        const uint64_t bag0 = base / a.chunks;
        const uint32_t local = (uint32_t)(base - bag0 * a.chunks) + threadIdx.x;
        const uint64_t bag = bag0 + local / a.chunks;
        const Piece<V> piece(local % a.chunks, a.t.dim);
        uint64_t begin, end;
        bag_range(a.b, bag, &begin, &end);
        float acc[V] = {};
        add_rows<E, V>(a, begin, end, 1, piece, acc);
        store_out<O, V>(a, bag, piece, acc);
    }
}

// Few bags, long ones: a workgroup per (bag, 64 pieces), whose 16 waves take every 16th position each and join their
// sums in LDS, in the order of the waves.
template <typename E, typename O, int V>
__global__ __launch_bounds__(1024) void lookup_split_kernel(LookupArgs a) {
    __shared__ float part[16][V][64];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t blocks = (a.chunks + 63) / 64;
    const uint64_t bag = blockIdx.x / blocks;
    const uint32_t chunk = blockIdx.x % blocks * 64 + lane;
    uint64_t begin, end;
    bag_range(a.b, bag, &begin, &end);
    float acc[V] = {};
    const Piece<V> piece(min(chunk, a.chunks - 1), a.t.dim);
    if (chunk < a.chunks) add_rows<E, V>(a, begin + wave, end, 16, piece, acc);
#pragma unroll
    for (int v = 0; v < V; ++v) part[wave][v][lane] = acc[v];
    __syncthreads();
    if (wave || chunk >= a.chunks) return;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        float sum = 0;
        for (int w = 0; w < 16; ++w) sum += part[w][v][lane];
        acc[v] = sum;
    }
    store_out<O, V>(a, bag, piece, acc);
}

template <typename E, typename O, int V>
hipError_t run_lookup(LookupArgs a, hipStream_t stream) {
    a.chunks = (a.t.dim + V - 1) / V;
    const uint64_t threads = a.b.n_bags * a.chunks;
    const uint64_t blocks = (a.chunks + 63) / 64;
    // With one thread per piece a bag of n ids takes n / 4 trips to memory; fewer threads than an eighth of what the
    // card holds (512 K) leave most of it idle meanwhile. Splitting pays once a bag has more ids than the 16 waves (4 bags of
    // up to 500, 768 f32: 13 us, 130 without; 64 of up to 40, 768 bf16: 5.4 and 14).
    if (threads < 65536 && a.b.n_ids > 16 * a.b.n_bags && a.b.n_bags * blocks < (1u << 20))
        lookup_split_kernel<E, O, V><<<(uint32_t)(a.b.n_bags * blocks), 1024, 0, stream>>>(a);
    else
        lookup_kernel<E, O, V><<<(uint32_t)std::min<uint64_t>((threads + 255) / 256, 1u << 20), 256, 0, stream>>>(a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_lookup(const Table& t, const Bags& b, void* out, int32_t out_dtype, uint64_t out_stride,
                         hipStream_t stream) {
    LookupArgs a{t, b, out, out_stride, 0};
    if (!b.n_bags) return hipSuccess;
    if (t.dtype == VS_F32)
        return out_dtype == VS_F32 ? run_lookup<float, float, 4>(a, stream) : run_lookup<float, bf16, 4>(a, stream);
    return out_dtype == VS_F32 ? run_lookup<bf16, float, 8>(a, stream) : run_lookup<bf16, bf16, 8>(a, stream);
}

// ---- gradients -----------------------------------------------------------------------------

namespace {

// The n (row, position) pairs are sorted by row, positions ascending within a row, so that a row's sum is a run of
// neighbours, taken in one order. Positions outside every bag and ids without a row get the row n_rows and come last.
constexpr uint32_t SMALL = 2048;      // ids of the one-kernel sort
constexpr uint32_t TILE = 1024;       // keys of a workgroup in a pass of the long sort
constexpr uint32_t RUN = 64;          // sorted entries that one thread sums before it hands over

struct GradArgs {
    const void* grad_out;
    uint64_t grad_stride;
    uint32_t dim, chunks;
    Bags b;
    uint64_t n_rows;
    uint32_t n;        // ids
    uint32_t n_runs;   // pieces of RUN sorted entries
    // workspace
    uint32_t* keys[2];
    uint32_t* places[2];  // after the sort, behind its last pass' keys: bag (places) and weight (keys) of each entry
    uint32_t* hist;
    uint32_t* totals;
    uint32_t* bag_at;  // [n] the bag of each position
    uint32_t* heads;   // first entries of runs, counted per TILE of sorted entries
    uint32_t* handed;  // [n_runs] number of the run that each piece hands over at its end
    float* partial;    // [n_runs][2][chunks * V]
    RowGrads out;
};

__device__ __forceinline__ uint32_t bag_of(const Bags& b, uint32_t p) {
    if (!b.offsets) return p < b.n_bags ? p : NONE;
    if (!b.n_bags || p < b.offsets[0] || p >= b.offsets[b.n_bags]) return NONE;
    uint64_t lo = 0, hi = b.n_bags;  // the last bag whose offset is <= p
    while (hi - lo > 1) {
        const uint64_t mid = (lo + hi) / 2;
        if (b.offsets[mid] <= p)
            lo = mid;
        else
            hi = mid;
    }
    return (uint32_t)lo;
}

__device__ __forceinline__ uint32_t key_of(const GradArgs& a, uint32_t p) {
    const uint32_t id = a.b.ids[p];
    if (id >= a.n_rows) return (uint32_t)a.n_rows;
    if (a.b.offsets && (p < a.b.offsets[0] || p >= a.b.offsets[a.b.n_bags])) return (uint32_t)a.n_rows;
    return !a.b.offsets && p >= a.b.n_bags ? (uint32_t)a.n_rows : id;
}

// Up to SMALL ids: entry p's place is the number of entries that sort before it, counted against all of them in LDS,
// four threads an entry and four comparisons a read. One launch, where the passes below are nine. The offsets are
// searched in LDS too: from memory, each step of a search would wait for the one before it. 160 ids: 5 us and the sums 5,
// by the passes 72 in all; 2000 ids: 24 and 13, by the passes 105.
__global__ __launch_bounds__(256) void rank_sort_kernel(GradArgs a) {
    __shared__ __align__(16) uint32_t keys[SMALL];
    __shared__ uint32_t offsets[SMALL + 1];
    const bool near = a.b.offsets && a.b.n_bags <= SMALL;
    if (near)
        for (uint32_t i = threadIdx.x; i <= a.b.n_bags; i += 256) offsets[i] = a.b.offsets[i];
    const uint32_t padded = (a.n + 15) / 16 * 16;
    for (uint32_t i = threadIdx.x; i < padded; i += 256) keys[i] = i < a.n ? key_of(a, i) : NONE;
    __syncthreads();
    const uint32_t p = blockIdx.x * 64 + (threadIdx.x >> 2), quarter = threadIdx.x & 3;
    const uint32_t key = p < a.n ? keys[p] : NONE;
    uint32_t place = 0;
#pragma unroll 4
    for (uint32_t i = quarter * 4; i < padded; i += 16) {
        const u32x4 k = *reinterpret_cast<const u32x4*>(keys + i);
#pragma unroll
        for (int j = 0; j < 4; ++j) place += k[j] < key || (k[j] == key && i + j < p);
    }
    place += __shfl_xor(place, 1);
    place += __shfl_xor(place, 2);
    if (p >= a.n || quarter) return;
    Bags b = a.b;
    if (near) b.offsets = offsets;
    a.keys[0][place] = key;
    a.places[1][place] = key < a.n_rows ? bag_of(b, p) : 0;
    reinterpret_cast<float*>(a.keys[1])[place] = a.b.weights ? a.b.weights[p] : 1.0f;
}

// A stable pass by 8 bits (328 thousand ids: 19 us, of launches mostly): counts of each digit in each tile ...
__global__ __launch_bounds__(256) void sort_count_kernel(GradArgs a, int pass, uint32_t n_tiles) {
    __shared__ uint32_t hist[256];
    hist[threadIdx.x] = 0;
    __syncthreads();
    const uint32_t* keys = a.keys[pass & 1];
    const uint32_t begin = blockIdx.x * TILE, end = min(begin + TILE, a.n);
    for (uint32_t i = begin + threadIdx.x; i < end; i += 256) {
        const uint32_t key = pass ? keys[i] : key_of(a, i);
        atomicAdd(&hist[key >> (8 * pass) & 255], 1u);  // counts: the order does not matter
    }
    __syncthreads();
    a.hist[(uint64_t)threadIdx.x * n_tiles + blockIdx.x] = hist[threadIdx.x];
}

// ... their sums over the tiles before, one workgroup per digit ...
__global__ __launch_bounds__(256) void sort_scan_kernel(GradArgs a, uint32_t n_tiles) {
    __shared__ uint32_t wave_sum[4];
    uint32_t* h = a.hist + (uint64_t)blockIdx.x * n_tiles;
    uint32_t before = 0;
    for (uint32_t base = 0; base < n_tiles; base += 256) {
        const uint32_t i = base + threadIdx.x;
        const uint32_t x = i < n_tiles ? h[i] : 0;
        uint32_t total;
        const uint32_t ex = block_exclusive(x, wave_sum, &total);
        if (i < n_tiles) h[i] = before + ex;
        before += total;
    }
    if (!threadIdx.x) a.totals[blockIdx.x] = before;
}

// ... and every key to its place: a tile's keys in rounds of 256, in order; within a wave the rank among equal digits
// comes from eight ballots.
__global__ __launch_bounds__(256) void sort_scatter_kernel(GradArgs a, int pass, uint32_t n_tiles) {
    __shared__ uint32_t next[256], counts[4][256], wave_sum[4];
    const uint32_t t = threadIdx.x, lane = t & 63, wave = t >> 6;
    uint32_t total;
    next[t] = block_exclusive(a.totals[t], wave_sum, &total) + a.hist[(uint64_t)t * n_tiles + blockIdx.x];
    const uint32_t *keys = a.keys[pass & 1], *places = a.places[pass & 1];
    uint32_t *out_keys = a.keys[~pass & 1], *out_places = a.places[~pass & 1];
    const uint32_t begin = blockIdx.x * TILE, end = min(begin + TILE, a.n);
    for (uint32_t base = begin; base < end; base += 256) {
#pragma unroll
        for (int w = 0; w < 4; ++w) counts[w][t] = 0;
        __syncthreads();
        const uint32_t i = base + t;
        const bool in = i < end;
        const uint32_t key = !in ? 0 : pass ? keys[i] : key_of(a, i);
        const uint32_t digit = key >> (8 * pass) & 255;
        uint64_t same = __ballot(in);
#pragma unroll
        for (int bit = 0; bit < 8; ++bit) {
            const bool one = digit >> bit & 1;
            const uint64_t m = __ballot(one);
            same &= one ? m : ~m;
        }
        const uint32_t rank = __popcll(same & ((1ull << lane) - 1));
        if (in && !rank) counts[wave][digit] = __popcll(same);
        __syncthreads();
        if (in) {
            uint32_t at = next[digit] + rank;
            for (uint32_t w = 0; w < wave; ++w) at += counts[w][digit];
            out_keys[at] = key;
            out_places[at] = pass ? places[i] : i;
        }
        __syncthreads();
        next[t] += counts[0][t] + counts[1][t] + counts[2][t] + counts[3][t];
    }
}

// Whether sorted entry i is the first of its row's run.
__device__ __forceinline__ bool is_head(const GradArgs& a, const uint32_t* keys, uint32_t i) {
    return keys[i] < a.n_rows && (!i || keys[i - 1] != keys[i]);
}

// The bag of every position (neighbours walk the same way through the offsets, so one line serves a wave at each step;
// looked up after the sort, every lane would walk its own).
__global__ __launch_bounds__(256) void map_bags_kernel(GradArgs a) {
    const uint32_t p = blockIdx.x * 256 + threadIdx.x;
    if (p < a.n) a.bag_at[p] = bag_of(a.b, p);
}

// After the last pass: each entry's bag and weight, so that the sums read them in order, and the heads of each tile.
__global__ __launch_bounds__(256) void settle_kernel(GradArgs a, int side) {
    __shared__ uint32_t wave_sum[4];
    uint32_t n = 0;
    const uint32_t begin = blockIdx.x * TILE, end = min(begin + TILE, a.n);
    const uint32_t *keys = a.keys[side], *places = a.places[side];
#pragma unroll
    for (uint32_t k = 0; k < TILE; k += 256) {
        const uint32_t i = begin + k + threadIdx.x;
        if (i >= end) break;
        n += is_head(a, keys, i);
        const uint32_t p = places[i];
        a.places[!side][i] = keys[i] < a.n_rows ? a.bag_at[p] : 0;
        reinterpret_cast<float*>(a.keys[!side])[i] = a.b.weights ? a.b.weights[p] : 1.0f;
    }
    uint32_t total;
    block_exclusive(n, wave_sum, &total);
    if (!threadIdx.x) a.heads[blockIdx.x] = total;
}

// Heads before sorted entry `at`, by a whole workgroup of 256.
__device__ uint32_t heads_before(const GradArgs& a, const uint32_t* keys, uint32_t at, uint32_t* wave_sum) {
    uint32_t n = 0;
    const uint32_t tile = at / TILE;
    if (a.heads)
        for (uint32_t i = threadIdx.x; i < tile; i += 256) n += a.heads[i];
    for (uint32_t i = (a.heads ? tile * TILE : 0) + threadIdx.x; i < at; i += 256) n += is_head(a, keys, i);
    uint32_t total;
    block_exclusive(n, wave_sum, &total);
    return total;
}

template <typename O, int V>
__device__ __forceinline__ void store_row(const GradArgs& a, uint32_t row, uint32_t compact, const Piece<V>& piece, const float (&acc)[V]) {
    O* out = static_cast<O*>(a.out.rows) + (uint64_t)(a.out.unique ? compact : row) * a.out.stride;
    Pack<O, V> p;
    if (!a.out.unique) p = load_piece<O, V>(out, piece, a.dim);  // a column of a row belongs to one thread: a plain addition
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const float x = acc[v] * a.b.scale;
        p.e[v] = from_f32<O>(a.out.unique ? x : x + to_f32(p.e[v]));
    }
    store_piece<O, V>(out, piece, a.dim, p, !a.out.unique);
}

// Up to SMALL ids: a workgroup per (sorted entry, 64 pieces). The ones at a run's head sum the run, a quarter in each
// of four waves.
template <typename E, typename O, int V>
__global__ __launch_bounds__(256) void sum_small_kernel(GradArgs a) {
    __shared__ float part[4][V][64];
    __shared__ uint32_t wave_sum[4];
    const uint32_t *keys = a.keys[0], *bags = a.places[1];
    const float* weights = reinterpret_cast<const float*>(a.keys[1]);
    const uint32_t i = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t chunk = blockIdx.y * 64 + lane;
    if (!blockIdx.y && i == a.n - 1 && a.out.count) {
        const uint32_t n = heads_before(a, keys, a.n, wave_sum);
        if (!threadIdx.x) *a.out.count = n;
    }
    if (!is_head(a, keys, i)) return;
    const uint32_t row = keys[i];
    uint32_t mine = 0, length;  // of the run
    for (uint32_t j = i + threadIdx.x; j < a.n; j += 256) mine += keys[j] == row;
    block_exclusive(mine, wave_sum, &length);
    const uint32_t end = i + length;
    const uint32_t compact = a.out.unique ? heads_before(a, keys, i, wave_sum) : 0;
    if (a.out.unique && !blockIdx.y && !threadIdx.x) a.out.unique[compact] = row;
    float acc[V] = {};
    if (chunk < a.chunks) {
        const E* g = static_cast<const E*>(a.grad_out);
#pragma unroll 4
        for (uint32_t j = i + wave; j < end; j += 4) {
            const Pack<E, V> x = load_piece<E, V>(g + (uint64_t)bags[j] * a.grad_stride, Piece<V>(chunk, a.dim), a.dim);
#pragma unroll
            for (int v = 0; v < V; ++v) acc[v] = __builtin_fmaf(weights[j], to_f32(x.e[v]), acc[v]);
        }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) part[wave][v][lane] = acc[v];
    __syncthreads();
    if (wave || chunk >= a.chunks) return;
#pragma unroll
    for (int v = 0; v < V; ++v) acc[v] = part[0][v][lane] + part[1][v][lane] + part[2][v][lane] + part[3][v][lane];
    store_row<O, V>(a, row, compact, Piece<V>(chunk, a.dim), acc);
}

// Many ids: one thread per (RUN sorted entries, V columns) walks its entries in order, eight gradients in flight. A
// row's run that lies within them is stored; what belongs to a run that began before or goes on behind is handed over
// in `partial`: [0] the run that was open at the first entry, [1] the one that is still open at the last (a run
// through all of them: [0] alone). 328 thousand gradients of 768 bf16, summed to 190 thousand f32 rows: 214 us, 5.1 TB/s of
// what is read (from cache) and written; entries are walked in order, so a thread waits for the eight it has asked for.
template <typename E, typename O, int V>
__global__ __launch_bounds__(256) void sum_runs_kernel(GradArgs a, int side) {
    constexpr int U = 8;
    __shared__ uint32_t wave_sum[4], heads_in[256];
    const uint32_t *keys = a.keys[side], *bags = a.places[!side];
    const float* weights = reinterpret_cast<const float*>(a.keys[!side]);
    const uint64_t first = (uint64_t)blockIdx.x * 256;
    const uint32_t run0 = (uint32_t)(first / a.chunks);
    const uint32_t local = (uint32_t)(first - (uint64_t)run0 * a.chunks) + threadIdx.x;
    const uint32_t run = run0 + local / a.chunks, chunk = local % a.chunks;
    uint32_t compact = 0;  // of the next head
    if (a.out.unique) {
        const uint32_t before = heads_before(a, keys, min(run0 * RUN, a.n), wave_sum);
        // the heads in each of the pieces that this workgroup's threads walk (256 at most: one of a thread each)
        uint32_t n = 0, total;
        const uint32_t r = run0 + threadIdx.x;
        if (r < a.n_runs && threadIdx.x <= 255 / a.chunks + 1)
            for (uint32_t i = r * RUN; i < min((r + 1) * RUN, a.n); ++i) n += is_head(a, keys, i);
        heads_in[threadIdx.x] = before + block_exclusive(n, wave_sum, &total);
        if (blockIdx.x == gridDim.x - 1) {
            const uint32_t all = heads_before(a, keys, a.n, wave_sum);
            if (!threadIdx.x) *a.out.count = all;
        }
        __syncthreads();
        compact = heads_in[run - run0];
    }
    if (run >= a.n_runs) return;
    const uint32_t begin = run * RUN, end = min(begin + RUN, a.n);
    const E* g = static_cast<const E*>(a.grad_out);
    const Piece<V> piece(chunk, a.dim);
    float* partial = a.partial + ((uint64_t)run * 2 * a.chunks + chunk) * V;
    uint32_t row = keys[begin];
    bool open = begin && keys[begin - 1] == row;  // the run began before
    float acc[V] = {};
    auto hand_over = [&](bool goes_on) {
        if (!open && a.out.unique && !chunk) a.out.unique[compact] = row;
        if (open || goes_on) {
            float* to = partial + (open ? 0 : (uint64_t)a.chunks * V);
#pragma unroll
            for (int v = 0; v < V; ++v) to[v] = acc[v];
        } else {
            store_row<O, V>(a, row, compact, piece, acc);
        }
        compact += !open;
        open = false;
    };
    for (uint32_t i = begin; i < end && row < a.n_rows; i += U) {
        uint32_t key[U];
        float w[U];
        Pack<E, V> x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t j = min(i + u, end - 1);
            key[u] = keys[j];
            w[u] = weights[j];
            x[u] = load_piece<E, V>(g + (uint64_t)bags[j] * a.grad_stride, piece, a.dim);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (i + u >= end) break;
            if (key[u] != row) {
                if (row < a.n_rows) hand_over(false);
                row = key[u];
#pragma unroll
                for (int v = 0; v < V; ++v) acc[v] = 0;
            }
#pragma unroll
            for (int v = 0; v < V; ++v) acc[v] = __builtin_fmaf(w[u], to_f32(x[u].e[v]), acc[v]);
        }
    }
    if (row >= a.n_rows) return;
    if (!chunk) a.handed[run] = compact;
    hand_over(end < a.n && keys[end] == row);
}

// The runs that were handed over (of 328 thousand ids: 32 us): a workgroup per (piece where one began, 64 pieces of
// columns); four waves take every fourth part each.
template <typename O, int V>
__global__ __launch_bounds__(256) void join_runs_kernel(GradArgs a, int side) {
    __shared__ float part[4][V][64];
    const uint32_t* keys = a.keys[side];
    const uint32_t run = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t begin = run * RUN, end = min(begin + RUN, a.n);
    if (end == a.n) return;
    const uint32_t row = keys[end];
    if (row >= a.n_rows || keys[end - 1] != row) return;
    if (begin && keys[begin] == row && keys[begin - 1] == row) return;  // began before
    uint32_t lo = run + 1, hi = a.n_runs;  // the last piece that begins with this row
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (keys[mid * RUN] == row)
            lo = mid;
        else
            hi = mid;
    }
    const uint32_t last = lo, compact = a.handed[run];
    const uint32_t chunk = blockIdx.y * 64 + lane;
    float acc[V] = {};
    if (chunk < a.chunks) {
        if (!wave) {
            const float* p = a.partial + (((uint64_t)run * 2 + 1) * a.chunks + chunk) * V;
#pragma unroll
            for (int v = 0; v < V; ++v) acc[v] = p[v];
        }
#pragma unroll 8
        for (uint32_t r = run + 1 + wave; r <= last; r += 4) {
            const float* p = a.partial + ((uint64_t)r * 2 * a.chunks + chunk) * V;
#pragma unroll
            for (int v = 0; v < V; ++v) acc[v] += p[v];
        }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) part[wave][v][lane] = acc[v];
    __syncthreads();
    if (wave || chunk >= a.chunks) return;
#pragma unroll
    for (int v = 0; v < V; ++v) acc[v] = part[0][v][lane] + part[1][v][lane] + part[2][v][lane] + part[3][v][lane];
    store_row<O, V>(a, row, compact, Piece<V>(chunk, a.dim), acc);
}

// A wave takes `span` neighbouring positions (64 at most: a lane looks up the row and the bag of each), four at a time:
// the products of each one's row with its bag's gradient, in pieces of V columns, joined over the lanes. 328 thousand of 768
// bf16: 133 us, 3.8 TB/s of rows and as much of gradients, which come from cache.
struct WeightArgs {
    Table t;
    Bags b;
    const void* grad_out;
    uint64_t grad_stride;
    float* out;
    uint32_t chunks, span;
};
template <typename E, typename G, int V>
__global__ __launch_bounds__(256) void weight_grads_kernel(WeightArgs a) {
    constexpr int U = 4;
    const uint32_t lane = threadIdx.x & 63, wave = uniform_u32(threadIdx.x >> 6);
    const uint64_t begin = ((uint64_t)blockIdx.x * 4 + wave) * a.span;
    if (begin >= a.b.n_ids) return;
    const uint32_t n = (uint32_t)min((uint64_t)a.span, a.b.n_ids - begin);
    uint32_t row = NONE, bag = NONE;
    if (lane < n) {
        row = row_of(a.t, a.b.ids[begin + lane]);
        bag = bag_of(a.b, (uint32_t)begin + lane);
        if (bag == NONE) row = NONE;
    }
    float result = 0;
    const E* rows = static_cast<const E*>(a.t.rows);
    const G* grads = static_cast<const G*>(a.grad_out);
    for (uint32_t i = 0; i < n; i += U) {
        uint32_t r[U], g[U];
        float sum[U] = {};
#pragma unroll
        for (int u = 0; u < U; ++u) {
            r[u] = (uint32_t)__builtin_amdgcn_readlane((int)row, (int)min(i + u, 63u));
            g[u] = (uint32_t)__builtin_amdgcn_readlane((int)bag, (int)min(i + u, 63u));
        }
        for (uint32_t c = lane; c < a.chunks; c += 64) {
            const Piece<V> piece(c, a.t.dim);
            Pack<E, V> x[U];
            Pack<G, V> y[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {  // (a position without a row reads row 0 and bag 0, and is not used)
                x[u] = load_piece<E, V>(rows + (uint64_t)(r[u] == NONE ? 0 : r[u]) * a.t.stride, piece, a.t.dim);
                y[u] = load_piece<G, V>(grads + (uint64_t)(r[u] == NONE ? 0 : g[u]) * a.grad_stride, piece, a.t.dim);
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const float s = __builtin_fmaf(to_f32(x[u].e[v]), to_f32(y[u].e[v]), sum[u]);
                    sum[u] = v >= (int)piece.skip ? s : sum[u];
                }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float total = wave_sum(sum[u]);
            if (lane == i + u) result = row == NONE ? 0.0f : total * a.b.scale;
        }
    }
    if (lane < n) a.out[begin + lane] = result;
}

template <typename E, typename O, int V>
hipError_t run_lookup_grad(GradArgs a, hipStream_t stream) {
    a.chunks = (a.dim + V - 1) / V;
    const uint32_t col_blocks = (a.chunks + 63) / 64;
    if (a.n <= SMALL) {
        a.heads = nullptr;
        rank_sort_kernel<<<(a.n + 63) / 64, 256, 0, stream>>>(a);
        sum_small_kernel<E, O, V><<<dim3(a.n, col_blocks), 256, 0, stream>>>(a);
        return hipGetLastError();
    }
    const uint32_t n_tiles = (a.n + TILE - 1) / TILE;
    int passes = 1;
    while (passes < 4 && a.n_rows >> (8 * passes)) ++passes;
    for (int pass = 0; pass < passes; ++pass) {
        sort_count_kernel<<<n_tiles, 256, 0, stream>>>(a, pass, n_tiles);
        sort_scan_kernel<<<256, 256, 0, stream>>>(a, n_tiles);
        sort_scatter_kernel<<<n_tiles, 256, 0, stream>>>(a, pass, n_tiles);
    }
    const int side = passes & 1;
    map_bags_kernel<<<(a.n + 255) / 256, 256, 0, stream>>>(a);
    settle_kernel<<<n_tiles, 256, 0, stream>>>(a, side);
    const uint64_t threads = (uint64_t)a.n_runs * a.chunks;
    sum_runs_kernel<E, O, V><<<(uint32_t)((threads + 255) / 256), 256, 0, stream>>>(a, side);
    join_runs_kernel<O, V><<<dim3(a.n_runs, col_blocks), 256, 0, stream>>>(a, side);
    return hipGetLastError();
}

uint64_t padded_dim(uint32_t dim) { return (dim + 7ull) / 8 * 8; }

}  // namespace

uint64_t lookup_grad_workspace_bytes(uint64_t n_ids, uint64_t n_rows, uint32_t dim) {
    const uint64_t n_tiles = (n_ids + TILE - 1) / TILE, n_runs = (n_ids + RUN - 1) / RUN;
    return 5 * round_up(n_ids * 4, 256) + round_up(n_tiles * 1024, 256) + 1024 + round_up(n_tiles * 4, 256) + round_up(n_runs * 4, 256) +
           (n_ids <= SMALL ? 0 : round_up(n_runs * 2 * padded_dim(dim) * 4, 256)) + 256;
}

hipError_t launch_lookup_grad(const void* grad_out, int32_t dtype, uint64_t grad_stride, uint32_t dim, const Bags& b,
                              uint64_t n_rows, void* workspace, const RowGrads& out, hipStream_t stream) {
    GradArgs a{};
    a.grad_out = grad_out;
    a.grad_stride = grad_stride;
    a.dim = dim;
    a.b = b;
    a.n_rows = n_rows;
    a.n = (uint32_t)b.n_ids;
    a.n_runs = (a.n + RUN - 1) / RUN;
    a.out = out;
    if (!a.n || !b.n_bags) {
        if (out.count) fill_u32(out.count, 1, 0u, stream);
        return hipGetLastError();
    }
    Carver w(workspace);
    for (int i = 0; i < 2; ++i) a.keys[i] = w.take<uint32_t>(a.n);
    for (int i = 0; i < 2; ++i) a.places[i] = w.take<uint32_t>(a.n);
    const uint32_t n_tiles = (a.n + TILE - 1) / TILE;
    a.hist = w.take<uint32_t>(256ull * n_tiles);
    a.totals = w.take<uint32_t>(256);
    a.bag_at = w.take<uint32_t>(a.n);
    a.heads = w.take<uint32_t>(n_tiles);
    a.handed = w.take<uint32_t>(a.n_runs);
    a.partial = w.take<float>(a.n <= SMALL ? 0 : (uint64_t)a.n_runs * 2 * padded_dim(dim));
    auto pick = [&](auto e, auto o) {
        using E = decltype(e);
        using O = decltype(o);
        constexpr int V = 16 / sizeof(E);
        return run_lookup_grad<E, O, V>(a, stream);
    };
    if (dtype == VS_F32) return out.dtype == VS_F32 ? pick(float{}, float{}) : pick(float{}, bf16{});
    return out.dtype == VS_F32 ? pick(bf16{}, float{}) : pick(bf16{}, bf16{});
}

hipError_t launch_lookup_grad_weights(const Table& t, const Bags& b, const void* grad_out, int32_t grad_dtype,
                                      uint64_t grad_stride, float* out, hipStream_t stream) {
    WeightArgs a{t, b, grad_out, grad_stride, out, 0, 0};
    if (!b.n_ids) return hipSuccess;
    if (!b.n_bags) {  // (nothing to multiply with)
        fill_u32(reinterpret_cast<uint32_t*>(out), b.n_ids, 0u, stream);
        return hipGetLastError();
    }
    // enough waves for every SIMD to hold eight first; then longer spans, which look more bags up at once
    a.span = (uint32_t)std::min<uint64_t>((b.n_ids + 8191) / 8192, 64);
    const uint32_t grid = (uint32_t)((b.n_ids + 4 * a.span - 1) / (4 * a.span));
    auto pick = [&](auto e, auto g) {
        using E = decltype(e);
        using G = decltype(g);
        constexpr int V = 16 / sizeof(E);
        a.chunks = (t.dim + V - 1) / V;
        weight_grads_kernel<E, G, V><<<grid, 256, 0, stream>>>(a);
        return hipGetLastError();
    };
    if (t.dtype == VS_F32) return grad_dtype == VS_F32 ? pick(float{}, float{}) : pick(float{}, bf16{});
    return grad_dtype == VS_F32 ? pick(bf16{}, float{}) : pick(bf16{}, bf16{});
}

}  // namespace learn
}  // namespace vs
