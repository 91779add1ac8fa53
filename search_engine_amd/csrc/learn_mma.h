// Products of tiles on the bf16 matrix cores: the loop that the cross entropy's four products share.
//
// A workgroup of eight waves makes a tile of M x N sums over k, 64 k at a time. Both operands' pieces of a step go from
// memory straight into LDS (16 bytes a lane, no registers), into a buffer that an earlier step has left, while the matrix
// cores work on another: one barrier a step. 64 KiB a step (256 x 256), twice, are 128 of the 160 KiB of a CU; smaller
// tiles, whose steps are over sooner than memory answers, have up to four buffers and load as many steps ahead.
//
// Operands come in three shapes:
//   Rows<R>  [R rows][64 k], k contiguous: read as one ds_read_b128 a fragment;
//   Cols<C>  [64 k][C columns], columns contiguous (the sum runs over memory rows): read with the transposing
//            ds_read_b64_tr_b16, four k x 16 columns per 16 lanes;
//   FloatCols<C>  the same of f32 elements, read one by one.
// All keep their 16-byte chunks rotated by XOR with the row, so that the lanes of a read fall on different banks.
//
// f32 operands are three bf16 planes: x = h + m + l exactly (8 + 8 + 8 bits), and a product takes the six steps hh, hm, mh,
// mm, hl, lh; what is left out (ml, lm, ll) is below 2^-23 of hh. Six steps on the bf16 cores are 2.7 times as fast as the
// f32 matrix instruction, whose rate is a sixteenth.
#pragma once
#include "learn_device.h"

namespace vs {
namespace learn {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void* lds_void;
typedef __attribute__((address_space(1))) const void* global_void;
typedef __attribute__((address_space(3))) s16x4* lds_s16x4;

struct f32x8 {
    f32x4 half[2];
};

constexpr uint32_t THREADS = 512;
constexpr uint32_t STEP = 64;  // k of a step

// A matrix of bf16 planes in memory; every row starts at a multiple of 16 bytes.
struct Planes {
    const char* base;
    uint64_t plane;        // bytes from one plane to the next
    uint32_t stride;       // bytes from one row to the next
    const uint32_t* list;  // row i is list[i]; null: i
    uint32_t rows;         // valid rows; those behind are zeros
    uint32_t chunks;       // 16-byte chunks of a row; those behind are zeros
};

// 16 bytes of every lane from memory to LDS, to `to` + 16 * lane. In assembly, because behind the builtin the compiler
// waits for every load under way before it reads LDS again (it takes the reads to need what the loads write), and a
// step's loads would no longer pass under the step before it. The instruction has no result register; what it wrote is
// waited for by hand, at step_barrier.
__device__ __forceinline__ void load_to_lds(const char* from, const char* to) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
                 :
                 : "v"((global_void)from), "s"(uniform_u32((uint32_t)(uintptr_t)(lds_void)to))
                 : "memory", "m0");
}
// My loads have written LDS, but for the last BEHIND loads and stores that I issued (there have to be so many at least: the
// counter of both falls in the order of their issue), and my reads of it are done, and so are everybody's.
template <int BEHIND = 0>
__device__ __forceinline__ void step_barrier() {
    constexpr int N = BEHIND > 63 ? 63 : BEHIND;
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | (N >> 4) << 14);  // vmcnt(N) lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// [R][64 k]: 128 bytes a row, chunk c of row r at place c ^ (r & 7).
template <int R, bool LISTED = false>
struct Rows {
    static constexpr int BYTES = R * 128;
    static constexpr int LOADS = R / 64;
    uint32_t index[LISTED ? LOADS : 1], next[LISTED ? LOADS : 1];  // rows in memory, of this tile and (as listed) the next
    uint32_t first, chunk;
    __device__ __forceinline__ void init() { chunk = (threadIdx.x & 7) ^ (threadIdx.x >> 3 & 7); }
    // The rows of the tile that starts at row `at`: reads the list, ahead of its use (nothing looks at what was read
    // until then, so nothing waits for it).
    __device__ __forceinline__ void peek(const Planes& p, uint32_t at) {
        if constexpr (LISTED)
#pragma unroll
            for (int i = 0; i < LOADS; ++i) next[i] = p.list[min(at + i * 64 + (threadIdx.x >> 3), p.rows - 1)];
    }
    __device__ __forceinline__ void aim(uint32_t at) {  // (at or behind the last row: zeros)
        first = at;
        if constexpr (LISTED)
#pragma unroll
            for (int i = 0; i < LOADS; ++i) index[i] = next[i];
    }
    // Piece i of the step's loads.
    __device__ __forceinline__ void load(int i, const Planes& p, uint32_t kstep, uint32_t plane, const char* zeros, char* lds) const {
        const uint32_t r = first + i * 64 + (threadIdx.x >> 3);
        const bool in = kstep * 8 + chunk < p.chunks && r < p.rows;
        const char* from = p.base + ((uint64_t)kstep * 128 + plane * p.plane) + ((uint64_t)(LISTED ? index[i] : r) * p.stride + chunk * 16);
        load_to_lds(in ? from : zeros, lds + uniform_u32(threadIdx.x >> 6) * 1024 + i * 8192);
    }
    // Lane's 8 k of fragment `t` (16 rows) in half `kk` of the step.
    __device__ __forceinline__ static bf16x8 read(const char* lds, uint32_t tile, int kk) {
        const uint32_t l = threadIdx.x & 63;
        return *reinterpret_cast<const bf16x8*>(lds + (tile * 16 + (l & 15)) * 128 + (((kk * 4 + (l >> 4)) ^ (l & 7)) * 16));
    }
    // The same of f32 elements, 32 of which are a row of LDS: a half of the step is a tile of its own.
    __device__ __forceinline__ static f32x8 read_f32(const char* lds, uint32_t tile, int kk) {
        const uint32_t l = threadIdx.x & 63;
        const char* row = lds + kk * BYTES + (tile * 16 + (l & 15)) * 128;
        f32x8 x;
        x.half[0] = *reinterpret_cast<const f32x4*>(row + (((l >> 4) * 2) ^ (l & 7)) * 16);
        x.half[1] = *reinterpret_cast<const f32x4*>(row + (((l >> 4) * 2 + 1) ^ (l & 7)) * 16);
        return x;
    }
};

// [64 k][C]: C * 2 bytes a k, chunk c of k at place c ^ turn(k).
template <int C, bool LISTED = false>
struct Cols {
    static constexpr int BYTES = C * 128;
    static constexpr int CHUNKS = C / 8;
    static constexpr int LOADS = CHUNKS / 8;
    static constexpr int APART = 512 / CHUNKS;  // k between two loads of a thread
    uint32_t index[LISTED ? LOADS : 1];
    uint32_t k0, chunk;
    __device__ __forceinline__ static uint32_t turn(uint32_t k) {
        return CHUNKS >= 16 ? (2 * (k & 3)) ^ (8 * (k >> 3 & 1)) : 2 * (k & 3);
    }
    __device__ __forceinline__ void init() {
        k0 = threadIdx.x / CHUNKS;
        chunk = (threadIdx.x % CHUNKS) ^ turn(k0);  // (the k of further loads are APART = 16, 32 apart: the same turn)
    }
    // The memory rows of the step whose first k is row `first` of `end`: reads the list, ahead of its use.
    __device__ __forceinline__ void peek(const Planes& p, uint32_t first, uint32_t end) {
        if constexpr (LISTED)
#pragma unroll
            for (int i = 0; i < LOADS; ++i) index[i] = p.list[min(first + k0 + i * APART, end - 1)];
    }
    __device__ __forceinline__ void load(int i, const Planes& p, uint32_t first, uint32_t end, uint32_t first_chunk, uint32_t plane,
                                         const char* zeros, char* lds) const {
        const uint32_t c = first_chunk + chunk, r = first + k0 + i * APART;
        const char* from = p.base + (plane * p.plane + c * 16ull) + (uint64_t)(LISTED ? index[i] : r) * p.stride;
        load_to_lds(r < end && c < p.chunks ? from : zeros, lds + uniform_u32(threadIdx.x >> 6) * 1024 + i * 8192);
    }
    __device__ __forceinline__ static bf16x8 read(char* lds, uint32_t tile, int kk) {
        const uint32_t l = threadIdx.x & 63, k = kk * 32 + (l >> 4) * 8 + (l >> 2 & 3);
        char* at = lds + k * (C * 2) + (((tile * 2 + (l >> 1 & 1)) ^ turn((l >> 4) * 8 + (l >> 2 & 3))) * 16) + (l & 1) * 8;
        union {
            s16x4 half[2];
            bf16x8 all;
        } x;
        x.half[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)at);
        x.half[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(at + 4 * (C * 2)));
        return x.all;
    }
};

// [64 k][C] of f32: C * 4 bytes a k, chunk c of k at place c ^ turn(k): the four groups of 16 lanes that read 16 columns
// of k, k + 8, k + 16 and k + 24 fall on different banks.
template <int C, bool LISTED = false>
struct FloatCols {
    static constexpr int BYTES = C * 256;
    static constexpr int CHUNKS = C / 4;
    static constexpr int LOADS = CHUNKS / 8;
    static constexpr int APART = 512 / CHUNKS;  // k between two loads of a thread
    static_assert(APART == 16 && CHUNKS >= 16);
    uint32_t index[LISTED ? LOADS : 1];
    uint32_t k0, chunk;
    __device__ __forceinline__ static uint32_t turn(uint32_t k) { return 4 * (k >> 3 & 3); }
    __device__ __forceinline__ void init() {
        k0 = threadIdx.x / CHUNKS;
        chunk = (threadIdx.x % CHUNKS) ^ turn(k0);
    }
    __device__ __forceinline__ void peek(const Planes& p, uint32_t first, uint32_t end) {
        if constexpr (LISTED)
#pragma unroll
            for (int i = 0; i < LOADS; ++i) index[i] = p.list[min(first + k0 + i * APART, end - 1)];
    }
    __device__ __forceinline__ void load(int i, const Planes& p, uint32_t first, uint32_t end, uint32_t first_chunk, const char* zeros,
                                         char* lds) const {
        const uint32_t c = first_chunk + (chunk ^ turn(i * APART)), r = first + k0 + i * APART;
        const char* from = p.base + c * 16ull + (uint64_t)(LISTED ? index[i] : r) * p.stride;
        load_to_lds(r < end && c < p.chunks ? from : zeros, lds + uniform_u32(threadIdx.x >> 6) * 1024 + i * 8192);
    }
    __device__ __forceinline__ static f32x8 read_f32(const char* lds, uint32_t tile, int kk) {
        const uint32_t l = threadIdx.x & 63, c = tile * 16 + (l & 15);
        const char* at = lds + (kk * 32 + (l >> 4) * 8) * (C * 4) + ((c / 4) ^ turn((l >> 4) * 8)) * 16 + c % 4 * 4;
        f32x8 x;
#pragma unroll
        for (int i = 0; i < 8; ++i) x.half[i / 4][i % 4] = *reinterpret_cast<const float*>(at + i * (C * 4));
        return x;
    }
};

// x = planes[0] + .. exactly, three bf16.
struct Split {
    uint16_t h, m, l;
};
__device__ __forceinline__ Split split(float x) {
    Split s;
    s.h = (uint16_t)bf16_bits(x);
    const float hv = __builtin_bit_cast(float, (uint32_t)s.h << 16);
    // beyond bf16's largest number the rounding gives an infinity; of an infinity, or a NaN, nothing is left to split
    const bool whole = !(__builtin_fabsf(hv) < __builtin_inff());
    if (whole && __builtin_fabsf(x) < __builtin_inff()) s.h = (uint16_t)(__builtin_bit_cast(uint32_t, x) >> 16);
    const float r = whole && !(__builtin_fabsf(x) < __builtin_inff()) ? 0.0f : x - __builtin_bit_cast(float, (uint32_t)s.h << 16);
    s.m = (uint16_t)bf16_bits(r);
    s.l = (uint16_t)bf16_bits(r - __builtin_bit_cast(float, (uint32_t)s.m << 16));
    return s;
}


// The planes of eight elements each, with packed conversions: five and a half instructions an element. `top`: the largest
// magnitude. Beyond the largest number of bf16 (an infinity, or near f32's largest) it takes split_all instead.
constexpr float SPLIT_TOP = 3.38953139e38f;
template <int N>
__device__ __forceinline__ void split_fast(const f32x8 (&x)[N], bf16x8 (&planes)[3][N], float* top) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    *top = 0;
#pragma unroll
    for (int n = 0; n < N; ++n) {
        u32x4 part[3];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float a = x[n].half[i / 2][i % 2 * 2], b = x[n].half[i / 2][i % 2 * 2 + 1];
            *top = __builtin_fmaxf(__builtin_fmaxf(*top, __builtin_fabsf(a)), __builtin_fabsf(b));
#pragma unroll
            for (int p = 0; p < 3; ++p) {
                const uint32_t both = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
                part[p][i] = both;
                a -= __builtin_bit_cast(float, both << 16);
                b -= __builtin_bit_cast(float, both & 0xFFFF0000);
            }
        }
#pragma unroll
        for (int p = 0; p < 3; ++p) planes[p][n] = __builtin_bit_cast(bf16x8, part[p]);
    }
}
template <int N>
__device__ __forceinline__ void split_all(const f32x8 (&x)[N], bf16x8 (&planes)[3][N]) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
        Pack<uint16_t, 8> part[3];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const Split s = split(x[n].half[i / 4][i % 4]);
            part[0].e[i] = s.h;
            part[1].e[i] = s.m;
            part[2].e[i] = s.l;
        }
#pragma unroll
        for (int p = 0; p < 3; ++p) planes[p][n] = __builtin_bit_cast(bf16x8, part[p]);
    }
}

// The products of a step: TM x TN fragments of 16 x 16 per wave, which start at fragments m0 and n0. Lane l holds rows
// (of A) 4 (l >> 4) + 0..3 and column (of B) l & 15 of each.
//
// A step is walked in phases of up to 16 matrix instructions, (half of k, half of A's fragments). Each phase first asks
// for the fragments of the next one, and issues a few of the loads of later steps: issued all at once, behind the
// barrier, they would queue up at the CU's one load path (16 cycles a piece) with the matrix cores idle. The step's one
// barrier stands before its LAST phase, whose fragments are in registers by then: behind it the next step's half of LDS is
// complete and this step's is free, and there is still a phase of products to issue while the first fragments of the
// next step and the loads of the step after it are under way.
template <typename A, typename B, int TM, int TN>
struct Engine {
    static constexpr int HALVES = TM >= 8 ? 2 : 1, PHASES = 2 * HALVES, MH = TM / HALVES;
    bf16x8 fa[2][MH], fb[2][TN];
    uint32_t m0, n0;

    __device__ __forceinline__ void ask(char* a, char* b, int phase) {
        const int kk = phase / HALVES, h = phase % HALVES;
#pragma unroll
        for (int m = 0; m < MH; ++m) fa[phase & 1][m] = A::read(a, m0 + h * MH + m, kk);
        if (h == 0)
#pragma unroll
            for (int n = 0; n < TN; ++n) fb[kk][n] = B::read(b, n0 + n, kk);
        __builtin_amdgcn_sched_barrier(0);
    }
    // (a, b): this step's operands in LDS; (next_a, next_b): the next one's. `under_way(phase)` issues loads, in the last
    // phase into this step's buffer. BEHIND: loads of later steps that were issued after the last of the next one's;
    // `stored`: and after those the STORES of a tile's end.
    template <int BEHIND, int STORES, typename F>
    __device__ __forceinline__ void step(char* a, char* b, char* next_a, char* next_b, f32x4 (&acc)[TM][TN], uint32_t stored, F&& under_way) {
#pragma unroll
        for (int p = 0; p < PHASES; ++p) {
            const int kk = p / HALVES, h = p % HALVES;
            if (p + 1 < PHASES) {
                ask(a, b, p + 1);
            } else {
                if (STORES && stored)
                    step_barrier<BEHIND + STORES>();
                else
                    step_barrier<BEHIND>();
                ask(next_a, next_b, 0);
            }
            under_way(p);
#pragma unroll
            for (int m = 0; m < MH; ++m)
#pragma unroll
                for (int n = 0; n < TN; ++n)
                    acc[h * MH + m][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[p & 1][m], fb[kk][n], acc[h * MH + m][n], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
};

// f32 products with all six steps of planes at once: of the one operand, which many tiles share, the planes P (P::BYTES
// apart) are in LDS, of the other the f32 elements themselves, X, which the wave splits as it reads them. TP x TX
// fragments; P_FIRST: P's rows are the rows of the result. The largest product has a sum of its own, so that its f32
// roundings are not taken again with each of the smaller ones.
template <typename P, typename X, int TP, int TX, bool P_FIRST>
struct SplitEngine {
    static constexpr int TM = P_FIRST ? TP : TX, TN = P_FIRST ? TX : TP;
    bf16x8 fp[2][3][TP], planes[2][3][TX];
    f32x8 fx[TX];
    uint32_t p0, x0;

    // The fragments of the k that come next: half `kk` of P's step, and of X's the half `xk`.
    __device__ __forceinline__ void ask(char* p, int kk, char* x, int xk) {
#pragma unroll
        for (int t = 0; t < TX; ++t) fx[t] = X::read_f32(x, x0 + t, xk);
#pragma unroll
        for (int i = 0; i < 3; ++i)
#pragma unroll
            for (int t = 0; t < TP; ++t) fp[kk][i][t] = P::read(p + i * P::BYTES, p0 + t, kk);
        __builtin_amdgcn_sched_barrier(0);
    }
    // Before the first half step.
    __device__ __forceinline__ void start(char* p, char* x) {
        ask(p, 0, x, 0);
        split_all(fx, planes[0]);
    }
    // The products of half KK of a step. `wait` lets everybody's loads of the next half have come; (p, x, xk) are that
    // one's; `under_way` issues loads. While the matrix cores multiply, the wave splits the next half.
    template <int KK, typename W, typename F>
    __device__ __forceinline__ void half(W&& wait, char* p, char* x, int xk, f32x4 (&large)[TM][TN], f32x4 (&small)[TM][TN], F&& under_way) {
        constexpr int PP[6] = {2, 0, 1, 1, 0, 0}, PX[6] = {0, 2, 1, 0, 1, 0};
        wait();
        ask(p, KK ^ 1, x, xk);
        under_way();
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int c = 0; c < 6; ++c)
#pragma unroll
            for (int i = 0; i < TP; ++i)
#pragma unroll
                for (int j = 0; j < TX; ++j) {
                    const int m = P_FIRST ? i : j, n = P_FIRST ? j : i;
                    f32x4& sum = c == 5 ? large[m][n] : small[m][n];
                    sum = P_FIRST ? __builtin_amdgcn_mfma_f32_16x16x32_bf16(fp[KK][PP[c]][i], planes[KK][PX[c]][j], sum, 0, 0, 0)
                                  : __builtin_amdgcn_mfma_f32_16x16x32_bf16(planes[KK][PX[c]][j], fp[KK][PP[c]][i], sum, 0, 0, 0);
                }
        float top;
        split_fast(fx, planes[KK ^ 1], &top);
#pragma unroll
        for (int i = 0; i < 3; ++i)
#pragma unroll
            for (int t = 0; t < TX; ++t) asm("" : "+v"(planes[KK ^ 1][i][t]));  // (here, and not behind the branch below)
        __builtin_amdgcn_sched_group_barrier(8, 4, 0);
#pragma unroll
        for (int i = 4; i < 6 * TP * TX; ++i) {
            __builtin_amdgcn_sched_group_barrier(8, 1, 0);  // a matrix instruction (16 cycles, four of them to issue),
            __builtin_amdgcn_sched_group_barrier(2, 3, 0);  // and three others meanwhile
        }
        __builtin_amdgcn_sched_barrier(0);
        if (__any(top > SPLIT_TOP)) split_all(fx, planes[KK ^ 1]);
    }
};

// A wave's results on their way to memory. Lane l has, of row l & 15, the pieces m of PB bytes that lie at (4 m + (l >> 4))
// PB: stored from there, an instruction would touch 16 rows for 4 PB bytes each. Taken through LDS it writes rows of
// 4 M PB bytes (128 or 256) in whole. The 16-byte chunks of a row are rotated by XOR with it, as above.
template <int PB, int M>
struct Turn {
    static constexpr int ROW = 4 * M * PB, CHUNKS = ROW / 16, BYTES = 16 * ROW, STORES = BYTES / 1024;
    __device__ __forceinline__ static char* at(char* wave_lds, uint32_t row, uint32_t chunk) {
        return wave_lds + row * ROW + (chunk ^ (row & (CHUNKS - 1))) * 16;
    }
    template <typename P>
    __device__ __forceinline__ static void put(char* wave_lds, uint32_t lane, int m, const P& piece) {
        static_assert(sizeof(P) == PB);
        const uint32_t byte = (m * 4 + (lane >> 4)) * PB;
        *reinterpret_cast<P*>(at(wave_lds, lane & 15, byte / 16) + byte % 16) = piece;
    }
    // The lane's part of store j: 16 bytes of row(), at 16 chunk().
    __device__ __forceinline__ static uint32_t row(uint32_t lane, int j) { return (j * 64 + lane) / CHUNKS; }
    __device__ __forceinline__ static uint32_t chunk(uint32_t lane) { return lane % CHUNKS; }
    __device__ __forceinline__ static u32x4 get(char* wave_lds, uint32_t lane, int j) {
        return *reinterpret_cast<const u32x4*>(at(wave_lds, row(lane, j), chunk(lane)));
    }
};

// Buffers of a step's `bytes` that fit beside `others` in the LDS of a CU.
constexpr int buffers_of(int bytes, int others) { return std::min((160 * 1024 - others) / bytes, 4); }

// Which step of the products a side's loads have come to: plane pair c of 64 k block k of the workgroup's tile `tile`.
struct Cursor {
    uint32_t c, k, tile;
    // Whether the tile ended.
    __device__ __forceinline__ bool advance(uint32_t planes, uint32_t blocks, uint32_t stride) {
        if (++c < planes) return false;
        c = 0;
        if (++k < blocks) return false;
        k = 0;
        tile += stride;
        return true;
    }
};

// The steps of a product of planes: (plane of A, plane of B) of step c.
struct Steps {
    uint32_t n;
    uint32_t a, b;  // two bits a step
    __device__ __forceinline__ uint32_t plane_a(uint32_t c) const { return a >> (2 * c) & 3; }
    __device__ __forceinline__ uint32_t plane_b(uint32_t c) const { return b >> (2 * c) & 3; }
};

}  // namespace learn
}  // namespace vs
