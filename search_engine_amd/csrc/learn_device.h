// Helpers of the learning kernels: element types, packs of elements, sums over a wave and a workgroup, and the
// carving of a caller's workspace.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "vs_device.h"

namespace vs {
namespace learn {

struct bf16 {
    uint16_t bits;
};

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(bf16 x) { return __builtin_bit_cast(float, (uint32_t)x.bits << 16); }

// Round to nearest even; a NaN stays one.
__device__ __forceinline__ uint32_t bf16_bits(float x) {
    return __builtin_bit_cast(uint16_t, (__bf16)x);
}
template <typename O>
__device__ __forceinline__ O from_f32(float x) {
    if constexpr (sizeof(O) == 4)
        return x;
    else
        return O{(uint16_t)bf16_bits(x)};
}

// V elements that are loaded and stored at once.
template <typename E, int V>
struct alignas(sizeof(E) * V < 16 ? sizeof(E) * V : 16) Pack {
    E e[V];
};
// (as vectors: element by element the compiler would join a wide store with the narrow one of another branch, and
// take the narrow)
template <typename E, int V>
__device__ __forceinline__ Pack<E, V> load_pack(const E* p) {
    constexpr int N = sizeof(E) * V;
    if constexpr (N % 16 == 0) {
        Pack<E, V> x;
#pragma unroll
        for (int i = 0; i < N / 16; ++i) reinterpret_cast<u32x4*>(&x)[i] = reinterpret_cast<const u32x4*>(p)[i];
        return x;
    } else if constexpr (N == 8) {
        return __builtin_bit_cast(Pack<E, V>, *reinterpret_cast<const u32x2*>(p));
    } else {
        return *reinterpret_cast<const Pack<E, V>*>(p);
    }
}
template <typename E, int V>
__device__ __forceinline__ void store_pack(E* p, const Pack<E, V>& x) {
    constexpr int N = sizeof(E) * V;
    if constexpr (N % 16 == 0) {
#pragma unroll
        for (int i = 0; i < N / 16; ++i) reinterpret_cast<u32x4*>(p)[i] = reinterpret_cast<const u32x4*>(&x)[i];
    } else if constexpr (N == 8) {
        *reinterpret_cast<u32x2*>(p) = __builtin_bit_cast(u32x2, x);
    } else {
        *reinterpret_cast<Pack<E, V>*>(p) = x;
    }
}
// Four and two words at the address of an element of SIZE bytes.
template <int SIZE>
struct Words;
template <>
struct Words<4> {
    typedef uint32_t four __attribute__((ext_vector_type(4), aligned(4)));
    typedef uint32_t two __attribute__((ext_vector_type(2), aligned(4)));
};
template <>
struct Words<2> {
    typedef uint32_t four __attribute__((ext_vector_type(4), aligned(2)));
    typedef uint32_t two __attribute__((ext_vector_type(2), aligned(2)));
};

// V elements from any place that an element may have (the memory path takes vectors at any address; what it costs is
// a second line where one is crossed); from `limit` elements on, zeros, which are not read.
template <typename E, int V>
__device__ __forceinline__ Pack<E, V> load_any(const E* p, uint32_t limit) {
    constexpr int N = 16 / sizeof(E);  // elements of a vector
    using four = typename Words<sizeof(E)>::four;
    Pack<E, V> x = {};
    if (V % N == 0 && limit >= V) {
#pragma unroll
        for (int i = 0; i < V / N; ++i) reinterpret_cast<u32x4*>(&x)[i] = reinterpret_cast<const four*>(p)[i];
    } else if (V * sizeof(E) == 8 && limit >= V) {
        using two = typename Words<sizeof(E)>::two;
        *reinterpret_cast<u32x2*>(&x) = *reinterpret_cast<const two*>(p);
    } else {
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (v < (int)min(limit, (uint32_t)V)) x.e[v] = p[v];
    }
    return x;
}
// The same for a store; elements from `limit` on are left as they are.
template <typename E, int V>
__device__ __forceinline__ void store_any(E* p, const Pack<E, V>& x, uint32_t limit) {
    constexpr int N = 16 / sizeof(E);
    using four = typename Words<sizeof(E)>::four;
    if (V % N == 0 && limit >= V) {
#pragma unroll
        for (int i = 0; i < V / N; ++i) reinterpret_cast<four*>(p)[i] = reinterpret_cast<const u32x4*>(&x)[i];
    } else if (V * sizeof(E) == 8 && limit >= V) {
        using two = typename Words<sizeof(E)>::two;
        *reinterpret_cast<two*>(p) = *reinterpret_cast<const u32x2*>(&x);
    } else {
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (v < (int)min(limit, (uint32_t)V)) p[v] = x.e[v];
    }
}

// The c-th piece of V of a row's `dim` columns. The last one, where dim is no multiple of V, starts earlier and has its
// first `skip` columns in common with the one before: so it is one load like the others. (A row of less than V columns:
// one piece, column by column.)
template <int V>
struct Piece {
    uint32_t col, skip;
    __host__ __device__ __forceinline__ Piece(uint32_t c, uint32_t dim) {
        const uint32_t first = c * V;
        skip = first + V > dim && dim >= V ? first + V - dim : 0;
        col = first - skip;
    }
};
template <typename E, int V>
__device__ __forceinline__ Pack<E, V> load_piece(const E* row, const Piece<V>& piece, uint32_t dim) {
    if (dim >= V) return load_any<E, V>(row + piece.col, V);
    return load_any<E, V>(row, dim);
}
// The same for rows that a call reads once (they are not kept in the caches for what others would read again).
template <typename E, int V>
__device__ __forceinline__ Pack<E, V> load_piece_once(const E* row, const Piece<V>& piece, uint32_t dim) {
    if (dim < V) return load_any<E, V>(row, dim);
    static_assert(V * sizeof(E) == 16);
    using four = typename Words<sizeof(E)>::four;
    return __builtin_bit_cast(Pack<E, V>, __builtin_nontemporal_load(reinterpret_cast<const four*>(row + piece.col)));
}
// Stores a piece; the columns in common with the one before are left to that one if ONCE (an addition), or else get the
// same value twice.
template <typename E, int V>
__device__ __forceinline__ void store_piece(E* row, const Piece<V>& piece, uint32_t dim, const Pack<E, V>& x, bool once) {
    if (dim < V) {
        store_any<E, V>(row, x, dim);
    } else if (once && piece.skip) {
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (v >= (int)piece.skip) row[piece.col + v] = x.e[v];
    } else {
        store_any<E, V>(row + piece.col, x, V);
    }
}

// A value that the compiler takes for a new one: what is computed from it is not kept in registers across a loop.
__device__ __forceinline__ uint32_t afresh(uint32_t x) {
    asm volatile("" : "+v"(x));
    return x;
}

// The same for a value that all lanes share (a flag of a loop: the compiler would make a copy of the loop's body for each
// of its values, and run out of registers between them).
__device__ __forceinline__ uint32_t afresh_uniform(uint32_t x) {
    x = uniform_u32(x);
    asm volatile("" : "+s"(x));
    return x;
}

__device__ __forceinline__ float wave_sum(float v) { return wave_sum_f32(v); }
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int d = 32; d; d /= 2) v += __shfl_xor(v, d);
    return v;
}

// Sum of x over the threads before this one, and over all, in a workgroup of 256.
__device__ __forceinline__ uint32_t block_exclusive(uint32_t x, uint32_t* wave_sums /* 4, LDS */, uint32_t* total) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t in = x;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const uint32_t y = __shfl_up(in, d);
        if (lane >= (uint32_t)d) in += y;
    }
    __syncthreads();  // the sums of a call before this one have been read
    if (lane == 63) wave_sums[wave] = in;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (uint32_t w = 0; w < 4; ++w) {
        if (w < wave) before += wave_sums[w];
        all += wave_sums[w];
    }
    *total = all;
    return before + in - x;
}

inline uint64_t round_up(uint64_t x, uint64_t to) { return (x + to - 1) / to * to; }

// Hands out pieces of a workspace, each at a multiple of 256 bytes.
class Carver {
  public:
    explicit Carver(void* base) : at_((char*)round_up((uintptr_t)base, 256)) {}
    template <typename T>
    T* take(uint64_t n) {
        T* p = reinterpret_cast<T*>(at_);
        at_ += round_up(n * sizeof(T), 256);
        return p;
    }
    const char* at() const { return at_; }

  private:
    char* at_;
};

static __global__ __launch_bounds__(256) void fill_u32_kernel(uint32_t* p, uint64_t n, uint32_t value) {
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (uint64_t)gridDim.x * 256) p[i] = value;
}
// (a kernel and not hipMemsetAsync: the call may be recorded into a graph, whose memset nodes this library keeps out)
inline void fill_u32(uint32_t* p, uint64_t n, uint32_t value, hipStream_t stream) {
    if (n) fill_u32_kernel<<<(uint32_t)std::min<uint64_t>((n + 255) / 256, 4096), 256, 0, stream>>>(p, n, value);
}

}  // namespace learn
}  // namespace vs
