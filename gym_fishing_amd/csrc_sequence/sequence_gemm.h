// sequence_gemm.h -- the matrix product the loss is made of: a tile of sum_k A[m, k] B[n, k] per workgroup on the matrix cores,
// handed to an epilogue in registers.
//
// An operand is either k-contiguous (element (m, k) at m * ld + k) or k-major (at k * ld + m).  Both are brought to LDS by
// 16-byte loads that bypass the registers, 128 bytes of k (64 bf16, 32 f32) at a time into one of two buffers while the other is
// multiplied: one barrier per 128 bytes of k.  LDS positions are fixed by the load (lane * 16), so the global addresses are
// permuted instead: 16-byte chunk c of row m sits at c ^ (m / 2 % 8), and of a k-major row k the 32-byte (bf16) or 64-byte (f32)
// unit u at u ^ f(k), which spreads the 16 rows or four k's of one fragment read over all banks.  A k-contiguous fragment is one
// ds_read_b128; a k-major one is two transposing reads (ds_read_b64_tr_b16: four k's of a column to each lane) in bf16, four
// ds_read_b32 in f32.
//
// What the caller owes: k a multiple of the 128 bytes for k-contiguous operands (pad with zeros), rows readable up to their count
// (an index beyond is clamped to the last: the epilogue drops what comes of it); for k-major operands columns readable up to a
// multiple of 16 bytes.  k-major rows beyond `k_rows` are clamped too: the other operand must be zero there.
#pragma once
#include "sequence_common.h"

namespace fishing {
namespace seq {

template <typename T>
struct Operand {
    const T* p;
    int64_t ld;
    int64_t count;    // rows (k-contiguous) or readable columns (k-major) of m / n
    int64_t k_rows;   // k-major: rows that exist
};

// The tile of a workgroup: an XCD's workgroups stand on 8 x 4 tiles, not on 32 x 1, so that what they read of both operands stays in its L2
__device__ __forceinline__ void tile_of(int64_t id, int64_t tiles_m, int64_t tiles_n, int64_t& tm, int64_t& tn) {
    constexpr int64_t ROWS = 8;
    const int64_t run = xcd_run(id, tiles_m * tiles_n), group = uniform(run / (ROWS * tiles_n)), first = group * ROWS, in = run - first * tiles_n;
    const int64_t rows = tiles_m - first < ROWS ? tiles_m - first : ROWS;
    tn = uniform(in / rows);
    tm = first + in - tn * rows;
}

#define FISHING_LDS(p) ((__attribute__((address_space(3))) void*)(p))
#define FISHING_GLOBAL(p) ((const __attribute__((address_space(1))) void*)(p))

template <typename T, int BM, bool K_MAJOR, int THREADS>
struct Stage {
    static constexpr int BK = 128 / (int)sizeof(T), EPC = 16 / (int)sizeof(T);
    static constexpr int CHUNKS = BM * 8, STEPS = CHUNKS / THREADS;
    static constexpr int RB = BM * (int)sizeof(T), CPR = RB / 16;    // k-major: bytes, chunks of a row
    static_assert(CHUNKS % THREADS == 0, "whole waves of loads");

    static constexpr int UNITS = RB / (sizeof(T) == 2 ? 32 : 64);    // k-major: swizzled units of a row
    static __device__ __forceinline__ int unit_swizzle(int k) { return (sizeof(T) == 2 ? (k & 3) | ((k >> 3 & 1) << 2) : (k >> 2) & 3) & (UNITS - 1); }

    // The tile's corner is uniform (scalar registers); a lane's offset from it fits 32 bits
    static __device__ __forceinline__ void load(char* lds, const Operand<T>& o, int64_t m0, int64_t k0) {
        const int wave = threadIdx.x >> 6;
        const char* corner = (const char*)(K_MAJOR ? o.p + k0 * o.ld + m0 : o.p + m0 * o.ld + k0);
        const int pitch = (int)(o.ld * (int64_t)sizeof(T));
        const int64_t left_m = o.count - m0, left_k = o.k_rows - k0;
        const int last_m = left_m < BM ? (int)left_m - 1 : BM - 1, last_k = left_k < BK ? (int)left_k - 1 : BK - 1;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const int ci = s * THREADS + threadIdx.x;
            int at;
            if (!K_MAJOR) {
                const int m = ci >> 3, c = (ci & 7) ^ ((m >> 1) & 7);
                at = (m < last_m ? m : last_m) * pitch + c * 16;
            } else {
                constexpr int U = sizeof(T) == 2 ? 2 : 4;             // chunks of a swizzled unit
                const int k = ci / CPR, pos = ci % CPR;
                const int c = ((pos / U) ^ unit_swizzle(k)) * U + pos % U;
                at = (k < last_k ? k : last_k) * pitch + (c * EPC <= last_m ? c * 16 : 0);
            }
            __builtin_amdgcn_global_load_lds(FISHING_GLOBAL(corner + (uint32_t)at), FISHING_LDS(lds + (s * THREADS + wave * 64) * 16), 16, 0, 0);
        }
    }

    // the fragments of N tiles of 16 rows from m0 on, at fragment step s: bf16: k = 32 s + 8 (lane / 16) + 0 .. 7; f32: k = 16 s +
    // 4 (lane / 16) + 0 .. 3, one per matrix instruction
    typedef typename std::conditional<sizeof(T) == 2, bf16x8, f32x4>::type Frag;
    template <int N, int S>
    static __device__ __forceinline__ void read(const char* lds, int m0, Frag (&f)[N]) {
        const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
        if constexpr (!K_MAJOR) {
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const int m = m0 + n * 16 + i;
                f[n] = *(const Frag*)(lds + m * 128 + (((S * 4 + g) ^ ((m >> 1) & 7)) << 4));
            }
        } else if constexpr (sizeof(T) == 2) {
            // In assembly because the compiler takes the builtin for a reader of the buffer that is being filled and waits for the
            // loads in flight.  Four (two) tiles a block, the wait inside it.
            static_assert(N % 2 == 0, "blocks of two tiles");
            const int k = 8 * g + (i >> 2);
            const uint32_t row = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)lds + k * RB + ((i & 3) << 3);
            union Two {
                uint64_t h[2];
                bf16x8 f;
            };
            auto at = [&](int n) { return row + ((((m0 >> 4) + n) ^ unit_swizzle(k)) << 5); };
            if constexpr (N % 4 == 0) {
#pragma unroll
                for (int n = 0; n < N; n += 4) {
                    Two r[4];
                    asm volatile(
                        "ds_read_b64_tr_b16 %0, %8 offset:%12\n\tds_read_b64_tr_b16 %1, %8 offset:%13\n\t"
                        "ds_read_b64_tr_b16 %2, %9 offset:%12\n\tds_read_b64_tr_b16 %3, %9 offset:%13\n\t"
                        "ds_read_b64_tr_b16 %4, %10 offset:%12\n\tds_read_b64_tr_b16 %5, %10 offset:%13\n\t"
                        "ds_read_b64_tr_b16 %6, %11 offset:%12\n\tds_read_b64_tr_b16 %7, %11 offset:%13\n\t"
                        "s_waitcnt lgkmcnt(0)"
                        : "=&v"(r[0].h[0]), "=&v"(r[0].h[1]), "=&v"(r[1].h[0]), "=&v"(r[1].h[1]), "=&v"(r[2].h[0]), "=&v"(r[2].h[1]), "=&v"(r[3].h[0]), "=&v"(r[3].h[1])
                        : "v"(at(n)), "v"(at(n + 1)), "v"(at(n + 2)), "v"(at(n + 3)), "n"(S * 32 * RB), "n"((S * 32 + 4) * RB)
                        : "memory");
#pragma unroll
                    for (int x = 0; x < 4; ++x) f[n + x] = r[x].f;
                }
            } else {
#pragma unroll
                for (int n = 0; n < N; n += 2) {
                    Two r[2];
                    asm volatile(
                        "ds_read_b64_tr_b16 %0, %4 offset:%6\n\tds_read_b64_tr_b16 %1, %4 offset:%7\n\t"
                        "ds_read_b64_tr_b16 %2, %5 offset:%6\n\tds_read_b64_tr_b16 %3, %5 offset:%7\n\t"
                        "s_waitcnt lgkmcnt(0)"
                        : "=&v"(r[0].h[0]), "=&v"(r[0].h[1]), "=&v"(r[1].h[0]), "=&v"(r[1].h[1])
                        : "v"(at(n)), "v"(at(n + 1)), "n"(S * 32 * RB), "n"((S * 32 + 4) * RB)
                        : "memory");
                    f[n] = r[0].f;
                    f[n + 1] = r[1].f;
                }
            }
        } else {
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int k = 16 * S + 4 * g + j;
                    f[n][j] = *(const float*)(lds + k * RB + ((((m0 >> 4) + n) ^ unit_swizzle(k)) << 6) + (i << 2));
                }
        }
    }
};

__device__ __forceinline__ f32x4 mma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mma(f32x4 a, f32x4 b, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    return c;
}

// WM x WN waves; a wave owns BM / WM x BN / WN outputs, MT x NT matrix-core tiles: acc[i][j] holds rows (lane / 16) * 4 .. + 3 of
// tile i, column lane % 16 of tile j
template <typename T, int BM, int BN, int WM, int WN, bool A_MAJOR, bool B_MAJOR>
struct Gemm {
    static constexpr int THREADS = WM * WN * 64, MT = BM / WM / 16, NT = BN / WN / 16;
    static constexpr int BK = 128 / (int)sizeof(T), BYTES = (BM + BN) * 128;
    typedef Stage<T, BM, A_MAJOR, THREADS> SA;
    typedef Stage<T, BN, B_MAJOR, THREADS> SB;

    static __device__ __forceinline__ int row0() { return (threadIdx.x >> 6) / WN * (BM / WM); }
    static __device__ __forceinline__ int col0() { return (threadIdx.x >> 6) % WN * (BN / WN); }

    static __device__ __forceinline__ void stage(char* lds, const Operand<T>& a, int64_t m0, const Operand<T>& b, int64_t n0, int64_t k0) {
        SA::load(lds, a, m0, k0);
        SB::load(lds + BM * 128, b, n0, k0);
    }

    template <int S>
    static __device__ __forceinline__ void step(const char* lds, f32x4 (&acc)[MT][NT]) {
        // (one step's fragments at a time: the scheduler would fetch both and spill)
        __builtin_amdgcn_sched_barrier(0);
        typename SA::Frag fa[MT];
        typename SB::Frag fb[NT];
        SB::template read<NT, S>(lds + BM * 128, col0(), fb);
        SA::template read<MT, S>(lds, row0(), fa);
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[i][j] = mma(fa[i], fb[j], acc[i][j]);
    }

    static __device__ __forceinline__ void multiply(const char* lds, f32x4 (&acc)[MT][NT]) {
        step<0>(lds, acc);
        step<1>(lds, acc);
    }

    static __device__ __forceinline__ void landed() {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    }

    // k in [k_lo, k_hi), both multiples of BK
    static __device__ __forceinline__ void run(char* lds0, char* lds1, const Operand<T>& a, int64_t m0, const Operand<T>& b, int64_t n0, int64_t k_lo, int64_t k_hi,
                                               f32x4 (&acc)[MT][NT]) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        int left = (int)((k_hi - k_lo) / BK);
        if (left <= 0) return;
        stage(lds0, a, m0, b, n0, k_lo);
        landed();
        for (; left >= 2; left -= 2) {
            stage(lds1, a, m0, b, n0, k_lo + BK);
            multiply(lds0, acc);
            landed();
            k_lo += 2 * BK;
            if (left > 2) stage(lds0, a, m0, b, n0, k_lo);
            multiply(lds1, acc);
            landed();
        }
        if (left) multiply(lds0, acc);
    }

    // f(row, col, four values of rows row .. row + 3), tile-relative
    template <typename F>
    static __device__ __forceinline__ void each(f32x4 (&acc)[MT][NT], F f) {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) f(row0() + i * 16 + (lane >> 4) * 4, col0() + j * 16 + (lane & 15), acc[i][j]);
    }
};

}  // namespace seq
}  // namespace fishing
