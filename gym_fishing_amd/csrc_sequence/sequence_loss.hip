// sequence_loss.hip -- softmax cross entropy over the quota levels, in pieces of the levels, without keeping the logits.
//
//   z = h W^T        lse = log sum_v exp(z_v)        loss = lse - z_y        (0 where the target y is outside [0, levels))
//   dz = g (exp(z - lse) - [v == y])        dh = dz W        dW = dz^T h
//
// Forward: one product whose epilogue reduces each row's tile of logits to a maximum and a sum of exponentials; the tiles' pairs are
// joined afterwards.  Backward: per piece of the levels the logits are computed again and turned into dz (rounded to the operands'
// type: it is a factor of the two products that follow; sums stay in float32), kept for the piece as dz^T [level][row], where four
// rows of a lane's accumulator are one store, and multiplied twice: k-major for dh, k-contiguous for dW.  In bf16 that rounding of dz
// makes the gradients' error 1.4 times their own last rounding's; for a handful of rows, whose dh is mostly one term, up to twice.  As
// two terms dz would double both products: at 8192 x 32771 x 1024 another 2 x (283 + 256) us.
//
// 8192 x 32771 x 1024, bf16: forward 626 us (880 TFLOP/s), and a piece of 16384 levels dz 302 (910), dW 283 (970), dh 256 (1070); a
// library's product of that shape reaches 1100.  Bound by LDS: a step's 192 KiB of fragments (eight waves, 8 + 4 of 1 KiB, twice) and 64 KiB
// of staging take 2048 cycles of its 128 bytes, as many as the matrix cores need; the forward's and dz's exponentials come on top.
// float32 products run on the float32 matrix cores (5001 x 1009 x 200: 33 us each, the matrix cores 60% busy); as three bf16 terms, six
// products, 34 - 42.
// 103424 x 100 x 128, bf16: 20 us forward, 20 dz, 31 dh, 19 dW, 13 the clean copy of h: bound by bytes and launches.
#include "sequence_gemm.h"

namespace fishing {
namespace seq {

__device__ __forceinline__ int64_t target_of(const void* target, int bytes, int64_t row) {
    return bytes == 4 ? (int64_t)((const int32_t*)target)[row] : ((const int64_t*)target)[row];
}

constexpr float kLog2E = 1.4426950408889634f;
__device__ __forceinline__ float exp_fast(float x) { return __builtin_amdgcn_exp2f(x * kLog2E); }

// over the 16 lanes of a row of the accumulator (DPP rotations: no trip through LDS)
template <int N>
__device__ __forceinline__ float rotated(float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x120 | N, 0xf, 0xf, false));
}
__device__ __forceinline__ float max16(float x) {
    x = fmaxf(x, rotated<8>(x));
    x = fmaxf(x, rotated<4>(x));
    x = fmaxf(x, rotated<2>(x));
    return fmaxf(x, rotated<1>(x));
}
__device__ __forceinline__ float sum16(float x) {
    x += rotated<8>(x);
    x += rotated<4>(x);
    x += rotated<2>(x);
    return x + rotated<1>(x);
}

// Rows of `width` to rows of `padded`, zeros behind; rows of padded targets become zeros, whatever they hold (NaN times a zero dz is
// NaN).  The two operands' copies are one launch: the second's blocks come behind the first's.
template <typename T>
struct PadJob {
    const T* src;
    int64_t ld, rows;
    T* dst;
    const void* target;       // of the rows, or none
};

template <typename T>
__global__ void __launch_bounds__(256) pad_kernel(PadJob<T> first, PadJob<T> second, int64_t first_blocks, int32_t width, int32_t padded, int target_bytes, int64_t levels) {
    const bool behind = blockIdx.x >= first_blocks;
    const PadJob<T> job = behind ? second : first;
    const int64_t block = behind ? blockIdx.x - first_blocks : blockIdx.x, ld = job.ld, rows = job.rows;
    const T* src = job.src;
    T* dst = job.dst;
    const void* target = job.target;
    constexpr int V = vec_of<T>();
    const int per = padded / V;
    const int64_t at = block * 256 + threadIdx.x;
    const int64_t row = at / per;
    const int c = (int)(at - row * per) * V;
    if (row >= rows) return;
    bool there = true;
    if (target) {
        const int64_t y = target_of(target, target_bytes, row);
        there = y >= 0 && y < levels;
    }
    Pack<T, V> x;
    const T* from = src + row * ld + c;
    if (there && c + V <= width && ((uintptr_t)from & 15) == 0) {
        x = *(const Pack<T, V>*)from;
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) x.e[e] = there && c + e < width ? from[e] : from_f32<T>(0.0f);
    }
    *(Pack<T, V>*)(dst + row * padded + c) = x;
}

// ---- forward: top[part][row], sum[part][row] of BN / WN levels each; taken[row] = the target's logit ----
template <typename T, typename G, int BM, int BN>
__global__ void __launch_bounds__(G::THREADS, 2)
    loss_part_kernel(Operand<T> h, Operand<T> w, int64_t k, const void* target, int target_bytes, int64_t tiles_m, int64_t tiles_n, float* top, float* sum, float* taken) {
    __shared__ __attribute__((aligned(16))) char lds0[G::BYTES];
    __shared__ __attribute__((aligned(16))) char lds1[G::BYTES];
    int64_t tm, tn;
    tile_of(blockIdx.x, tiles_m, tiles_n, tm, tn);
    // the target's column in this tile, or -1; read behind the product's barriers
    __shared__ int column[BM];
    if (threadIdx.x < BM) {
        const int64_t row = tm * BM + threadIdx.x;
        const int64_t y = row < h.count ? target_of(target, target_bytes, row) - tn * BN : -1;
        column[threadIdx.x] = y >= 0 && y < BN ? (int)y : -1;
    }
    f32x4 acc[G::MT][G::NT];
    G::run(lds0, lds1, h, tm * BM, w, tn * BN, 0, k, acc);
    const int lane = threadIdx.x & 63;
    const int64_t left = w.count - tn * BN, rows_left = h.count - tm * BM, part = (tn * BN + G::col0()) / (G::NT * 16);
    const int levels_here = left < BN ? (int)left : BN, rows_here = rows_left < BM ? (int)rows_left : BM, col = G::col0() + (lane & 15);
    float *top_here = top + part * h.count + tm * BM, *sum_here = sum + part * h.count + tm * BM, *taken_here = taken + tm * BM;
    const bool whole = levels_here == BN;
#pragma unroll
    for (int i = 0; i < G::MT; ++i) {
        const int row = G::row0() + i * 16 + (lane >> 4) * 4;
        const int4 y = *(const int4*)&column[row];
        const int ys[4] = {y.x, y.y, y.z, y.w};
        float m[4], s[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            if (!whole) {
#pragma unroll
                for (int j = 0; j < G::NT; ++j) acc[i][j][r] = col + j * 16 < levels_here ? acc[i][j][r] : -INFINITY;
            }
            m[r] = acc[i][0][r];
#pragma unroll
            for (int j = 1; j < G::NT; ++j) m[r] = fmaxf(m[r], acc[i][j][r]);
            m[r] = max16(m[r]);
            const float from = m[r] == -INFINITY ? 0.0f : m[r];      // (a part wholly behind the last level: m = -inf, s = 0)
            s[r] = 0.0f;
#pragma unroll
            for (int j = 0; j < G::NT; ++j) s[r] += exp_fast(acc[i][j][r] - from);
            s[r] = sum16(s[r]);
#pragma unroll
            for (int j = 0; j < G::NT; ++j)
                if (ys[r] == col + j * 16) taken_here[row + r] = acc[i][j][r];
        }
        if ((lane & 15) == 0) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if (row + r < rows_here) {
                    top_here[row + r] = m[r];
                    sum_here[row + r] = s[r];
                }
            }
        }
    }
}

// x of a row's lanes made one by `op`, the same in all of them: R rows x L lanes, the rows side by side
template <int R, int L, typename F>
__device__ __forceinline__ float over_row(float x, float (&shared)[R * L / 64][R], F op) {
    if constexpr (L == 1) return x;
#pragma unroll
    for (int d = R; d < 64; d <<= 1) x = op(x, __shfl_xor(x, d));
    constexpr int WAVES = R * L / 64;
    if constexpr (WAVES > 1) {
        const int r = threadIdx.x % R;
        __syncthreads();
        if ((threadIdx.x & 63) < R) shared[threadIdx.x >> 6][r] = x;
        __syncthreads();
        x = shared[0][r];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) x = op(x, shared[w][r]);
    }
    return x;
}

// lse = top + log sum_p sum_p exp(top_p - top): lane p0 of a row takes parts p0, p0 + L, ...  First the maximum, then the sum, whose
// terms then do not wait for each other.  Many parts (few rows against many levels) take many lanes: 17 rows, 2050 parts: 7.1 us,
// pairs joined one after the other 11.3; 8192 rows, 513 parts: 8.8, 18
template <int R, int L>
__global__ void __launch_bounds__(R* L) loss_join_kernel(const float* top, const float* sum, const float* taken, const void* target, int target_bytes, int64_t rows,
                                                         int64_t levels, int parts, float* loss, float* lse) {
    __shared__ float shared[R * L / 64][R];
    const int r = threadIdx.x % R, p0 = threadIdx.x / R;
    const int64_t row = (int64_t)blockIdx.x * R + r, at = row < rows ? row : rows - 1;
    float m = -INFINITY, s = 0.0f;
#pragma unroll 8
    for (int p = p0; p < parts; p += L) m = fmaxf(m, top[(int64_t)p * rows + at]);
    m = over_row<R, L>(m, shared, [](float x, float y) { return fmaxf(x, y); });
    const float from = m == -INFINITY ? 0.0f : m;
#pragma unroll 8
    for (int p = p0; p < parts; p += L) s += sum[(int64_t)p * rows + at] * exp_fast(top[(int64_t)p * rows + at] - from);
    s = over_row<R, L>(s, shared, [](float x, float y) { return x + y; });
    if (p0 || row >= rows) return;
    const float l = m + logf(s);
    lse[row] = l;
    const int64_t t = target_of(target, target_bytes, row);
    loss[row] = t >= 0 && t < levels ? l - taken[row] : 0.0f;
}

// ---- backward: dz^T of a piece of the levels, [width padded to BN][ld rows]; zeros behind the rows and the levels ----
template <typename T, typename G, int BM, int BN>
__global__ void __launch_bounds__(G::THREADS, 2)
    loss_dz_kernel(Operand<T> h, Operand<T> w, int64_t k, const void* target, int target_bytes, int64_t levels, int64_t v0, int64_t tiles_m, int64_t tiles_n, const float* lse,
                   const float* g, T* dzt, int64_t ld) {
    __shared__ __attribute__((aligned(16))) char lds0[G::BYTES];
    __shared__ __attribute__((aligned(16))) char lds1[G::BYTES];
    int64_t tm, tn;
    tile_of(blockIdx.x, tiles_m, tiles_n, tm, tn);
    // per row of the tile, read behind the product's barriers: lse (infinite for a padded target: a share of zero), the loss's
    // gradient, the target's column or -1
    __shared__ float row_lse[BM], row_g[BM];
    __shared__ int row_y[BM];
    if (threadIdx.x < BM) {
        const int64_t row = tm * BM + threadIdx.x, t = row < h.count ? target_of(target, target_bytes, row) : -1;
        const bool there = t >= 0 && t < levels;
        const int64_t rel = t - v0 - tn * BN;
        row_lse[threadIdx.x] = there ? lse[row] : INFINITY;
        row_g[threadIdx.x] = there ? g[row] : 0.0f;
        row_y[threadIdx.x] = there && rel >= 0 && rel < BN ? (int)rel : -1;
    }
    f32x4 acc[G::MT][G::NT];
    G::run(lds0, lds1, h, tm * BM, w, v0 + tn * BN, 0, k, acc);
    const int lane = threadIdx.x & 63, col = G::col0() + (lane & 15);
    const int64_t left = levels - v0 - tn * BN, ld_left = ld - tm * BM;
    const int levels_here = left < BN ? (int)left : BN, ld_here = ld_left < BM ? (int)ld_left : BM;
    T* to = dzt + (tn * BN + col) * ld + tm * BM;
#pragma unroll
    for (int i = 0; i < G::MT; ++i) {
        const int row = G::row0() + i * 16 + (lane >> 4) * 4;
        if (row >= ld_here) continue;
        const f32x4 l = *(const f32x4*)&row_lse[row], gr = *(const f32x4*)&row_g[row];
        const int4 y4 = *(const int4*)&row_y[row];
        const int y[4] = {y4.x, y4.y, y4.z, y4.w};
#pragma unroll
        for (int j = 0; j < G::NT; ++j) {
            Pack<T, 4> x;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float p = exp_fast(acc[i][j][r] - l[r]) - (y[r] == col + j * 16 ? 1.0f : 0.0f);
                x.e[r] = from_f32<T>(l[r] == INFINITY || col + j * 16 >= levels_here ? 0.0f : gr[r] * p);
            }
            *(Pack<T, 4>*)(to + j * 16 * ld + row) = x;
        }
    }
}

// ---- out[n][m] (+)= sum_k A[m, k] B[n, k] over a share of k: float32 slabs (one per share, added to across pieces) or the type.  PADDED:
// rows n of padded targets are zeros, whatever A holds (their dz is zero, and zero times NaN is NaN) ----
struct Targets {
    const void* target;
    int bytes;
    int64_t levels;
};

template <typename T, typename O, typename G, int BM, int BN, bool PADDED>
__global__ void __launch_bounds__(G::THREADS, 2)
    product_kernel(Operand<T> a, Operand<T> b, int64_t k, int64_t share, int64_t m, int64_t n, int64_t tiles_m, int64_t tiles_n, bool add, O* out, int64_t ld, int64_t slab,
                   Targets y) {
    __shared__ __attribute__((aligned(16))) char lds0[G::BYTES];
    __shared__ __attribute__((aligned(16))) char lds1[G::BYTES];
    int64_t tm, tn;
    tile_of(blockIdx.x, tiles_m, tiles_n, tm, tn);
    const int64_t lo = blockIdx.y * share, hi = lo + share < k ? lo + share : k;
    __shared__ bool gone[PADDED ? BN : 1];                // read behind the product's barriers (an empty share has none, and sums of zero)
    if (PADDED && threadIdx.x < BN) {
        const int64_t row = tn * BN + threadIdx.x, t = row < n ? target_of(y.target, y.bytes, row) : -1;
        gone[threadIdx.x] = t < 0 || t >= y.levels;
    }
    f32x4 acc[G::MT][G::NT];
    G::run(lds0, lds1, a, tm * BM, b, tn * BN, lo, hi, acc);
    const int64_t left_n = n - tn * BN, left_m = m - tm * BM;
    const int n_here = left_n < BN ? (int)left_n : BN, m_here = left_m < BM ? (int)left_m : BM;
    O* to = out + blockIdx.y * slab + tn * BN * ld + tm * BM;
    const bool whole = (ld & 3) == 0 && (((uintptr_t)out) & (4 * sizeof(O) - 1)) == 0;
    G::each(acc, [&](int r, int c, f32x4 x) {
        if (c >= n_here || r >= m_here) return;
        if (PADDED && gone[c]) x = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        O* p = to + c * ld + r;
        if (whole && r + 4 <= m_here) {
            Pack<O, 4> y;
            if (add) y = *(const Pack<O, 4>*)p;
#pragma unroll
            for (int e = 0; e < 4; ++e) y.e[e] = from_f32<O>(add ? to_f32(y.e[e]) + x[e] : x[e]);
            *(Pack<O, 4>*)p = y;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (r + e < m_here) p[e] = from_f32<O>(add ? to_f32(p[e]) + x[e] : x[e]);
        }
    });
}

// out = the shares' slabs added in order: L lanes take every L-th slab, their sums are added in the lanes' order
template <typename T, int L>
__global__ void __launch_bounds__(256) slab_sum_kernel(const float* slabs, int64_t slab, int count, T* out, int64_t n) {
    constexpr int C = 256 / L;
    __shared__ f32x4 lane_sum[L][C];
    const int c = threadIdx.x % C, l = threadIdx.x / C;
    const int64_t at = ((int64_t)blockIdx.x * C + c) * 4;
    f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
    if (at < n) {                                         // (a slab is padded to whole quads)
#pragma unroll 8
        for (int i = l; i < count; i += L) s += *(const f32x4*)(slabs + i * slab + at);
    }
    if (L > 1) {
        lane_sum[l][c] = s;
        __syncthreads();
        if (l) return;
#pragma unroll
        for (int i = 1; i < L; ++i) s += lane_sum[i][c];
    }
    if (at >= n) return;
    if (at + 4 <= n && ((uintptr_t)(out + at) & (4 * sizeof(T) - 1)) == 0) {
        Pack<T, 4> y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y.e[e] = from_f32<T>(s[e]);
        *(Pack<T, 4>*)(out + at) = y;
    } else {
        for (int e = 0; e < 4 && at + e < n; ++e) out[at + e] = from_f32<T>(s[e]);
    }
}

template <typename T>
static int slab_sum(const float* slabs, int64_t slab, int64_t count, T* out, int64_t n, hipStream_t stream) {
    if (count >= 32) return launch(slab_sum_kernel<T, 16>, dim3((unsigned)ceil_div(n, 64)), dim3(256), stream, slabs, slab, (int)count, out, n);
    return launch(slab_sum_kernel<T, 1>, dim3((unsigned)ceil_div(n, 1024)), dim3(256), stream, slabs, slab, (int)count, out, n);
}

template <typename T>
__global__ void __launch_bounds__(256) zero_kernel(T* p, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) p[i] = from_f32<T>(0.0f);
}

// ---- the plan: tile sizes, pieces, shares ----
constexpr int64_t kCUs = 256;

// What a workgroup's tile of b x b outputs costs, us: a staged 128 bytes of k, and what surrounds the product (first load, epilogue).
// Measured on 8192 x 32771 x 1024 (b = 256: 16 steps, 42 us a tile in all), 103424 x 100 x 128 (128) and 5001 x 1009 x 200 (64, f32)
template <typename T>
static double step_us(int64_t b) {
    if (sizeof(T) == 2) return b == 256 ? 2.0 : b == 128 ? 0.7 : 0.25;
    return b == 256 ? 7.6 : b == 128 ? 1.9 : 0.5;
}
static double tile_us(int64_t b) { return b == 256 ? 10.0 : b == 128 ? 4.0 : 2.0; }

struct Tiling {
    int64_t b, shares, share;       // tile edge; how often k is split, and the split's elements of k
};

// the tile and the split of k that fill the chip's rounds of workgroups best; every split costs a float32 slab written and read
template <typename T>
static Tiling tiling(int64_t m, int64_t n, int64_t k, bool split) {
    const int64_t bk = 128 / (int64_t)sizeof(T), steps = ceil_div(k, bk);
    Tiling best{64, 1, steps * bk};
    double least = -1.0;
    for (int64_t b = 256; b >= 64; b >>= 1) {
        const int64_t tiles = ceil_div(m, b) * ceil_div(n, b);
        for (int64_t s = 1; s <= (split ? 1024 : 1) && s <= steps; s <<= 1) {
            const double each = tile_us(b) + step_us<T>(b) * (double)ceil_div(steps, s);
            const double us = (double)ceil_div(tiles * s, kCUs) * each + (s > 1 ? 4.0 + (double)(s * m * n) * 8e-6 / 4.0 : 0.0);
            if (least < 0.0 || us < least) {
                least = us;
                best = Tiling{b, s, ceil_div(steps, s) * bk};
            }
        }
    }
    best.shares = ceil_div(steps * bk, best.share);
    return best;
}

// f(an object of the tile's product type, its edge): the run-time edge made a type
template <typename T, int B, bool A_MAJOR, bool B_MAJOR>
struct TileType {
    typedef Gemm<T, B, B, 2, B == 256 ? 4 : 2, A_MAJOR, B_MAJOR> G;
    static constexpr int EDGE = B;
};
template <typename T, bool A_MAJOR, bool B_MAJOR, typename F>
static int with_tile(int64_t b, F&& f) {
    return b == 256 ? f(TileType<T, 256, A_MAJOR, B_MAJOR>{}) : b == 128 ? f(TileType<T, 128, A_MAJOR, B_MAJOR>{}) : f(TileType<T, 64, A_MAJOR, B_MAJOR>{});
}
static int64_t part_levels(int64_t b) { return b == 256 ? 64 : b / 2; }      // levels of a wave's columns

// The rows are walked in blocks, so that dz^T of a piece stays under 2^30 elements, the forward's pairs under 2^28 and dz^T's pitch
// (2^21 rows: at most 8 MiB) within a staged tile's 32-bit offsets
constexpr int64_t kBlockRows = (int64_t)1 << 21, kMaxPitch = (int64_t)1 << 23;

struct LossPlan {
    int64_t block, bk, dim_p, rows_p, piece;       // rows of a block; elements of a staged k step; padded depth and block; levels of a piece
    int64_t z;                                     // forward: tile edge
    int parts;
    Tiling dh;                              // of a whole piece; the last one's is made for its width
};

template <typename T>
static Tiling dw_tiling(const LossPlan& p, int64_t width, int64_t dim) { return tiling<T>(dim, width, p.rows_p, true); }

template <typename T>
static LossPlan loss_plan(int64_t rows, int64_t levels, int64_t dim, bool backward) {
    LossPlan p{};
    rows = rows > 0 ? rows : 1;
    p.bk = 128 / (int64_t)sizeof(T);
    p.dim_p = round_up(dim, p.bk);
    p.z = tiling<T>(rows, levels, dim, false).b;
    p.parts = (int)(ceil_div(levels, p.z) * (p.z / part_levels(p.z)));
    // A piece keeps dz^T for the two products: at most 24576 levels, at least 8192, and of those the width whose product for dW
    // fills its rounds of workgroups best (32771 levels, dim 1024: three pieces of 43 tiles left a third of the chip idle)
    p.piece = levels;
    if (levels > 16384) {
        double best = 0.0;
        const int64_t across = ceil_div(dim, 256);
        for (int64_t t = 96; t >= 32; --t) {
            const int64_t tiles = t * across, s = tiles < kCUs ? kCUs / tiles : 1;
            const double full = (double)(tiles * s) / (double)round_up(tiles * s, kCUs);
            if (full > best + 1e-9) {
                best = full;
                p.piece = t * 256;
            }
        }
        if (p.piece > levels) p.piece = levels;
    }
    const int64_t widest = backward ? (p.piece > p.dim_p ? p.piece : p.dim_p) : (p.parts > p.dim_p / 4 ? p.parts : p.dim_p / 4) * 4;
    p.block = (((int64_t)1 << 30) / widest) & ~(int64_t)255;
    p.block = p.block < 256 ? 256 : p.block > kBlockRows ? kBlockRows : p.block;
    p.block = p.block > rows ? rows : p.block;
    p.rows_p = round_up(p.block, p.bk);
    p.dh = tiling<T>(dim, p.block, p.piece, true);
    return p;
}

template <typename T>
struct LossWork {
    float *top = nullptr, *sum = nullptr, *taken = nullptr, *dh = nullptr, *dw = nullptr;
    T *h = nullptr, *w = nullptr, *dzt = nullptr;
    int64_t dh_slab = 0, dw_slab = 0, bytes = 0;
};

// the padded copies are counted whether the operands need them or not: the caller asks before the pointers are known
template <typename T>
static LossWork<T> loss_work(const LossPlan& p, int64_t rows, int64_t levels, int64_t dim, bool backward, void* at) {
    Carve c(at);
    LossWork<T> w;
    w.h = c.take<T>(p.block * p.dim_p);
    w.w = c.take<T>(levels * p.dim_p);
    if (backward) {
        w.dzt = c.take<T>(round_up(p.piece, 256) * p.rows_p);
        w.dh_slab = round_up(p.block * dim, 4);
        if (p.dh.shares > 1 || p.piece < levels) w.dh = c.take<float>(p.dh.shares * w.dh_slab);
        const int64_t last = levels % p.piece, a = dw_tiling<T>(p, p.piece, dim).shares, b = last ? dw_tiling<T>(p, last, dim).shares : 1;
        const int64_t slabs_a = a > 1 ? a * round_up(p.piece * dim, 4) : 0, slabs_b = b > 1 ? b * round_up(last * dim, 4) : 0;
        // several blocks of rows add to slabs of all levels, one block's pieces share slabs of their own levels
        w.dw_slab = p.block < rows ? round_up(levels * dim, 4) : 0;
        w.dw = c.take<float>(w.dw_slab ? a * w.dw_slab : slabs_a > slabs_b ? slabs_a : slabs_b);
    } else {
        w.top = c.take<float>(p.block * p.parts);
        w.sum = c.take<float>(p.block * p.parts);
        w.taken = c.take<float>(p.block);
    }
    w.bytes = c.used + 256;
    return w;
}

static int loss_check(int32_t dtype, int64_t rows, int64_t levels, int64_t dim) {
    if (dtype != FISHING_DTYPE_F32 && dtype != FISHING_DTYPE_BF16) return FISHING_ERR_UNSUPPORTED;
    if (rows < 0 || rows > 0x7fffffff || levels < 1 || levels > 0x7ffffff || dim < 1 || dim > 65536) return FISHING_ERR_SIZE;
    if (levels * round_up(dim, 64) > (int64_t)1 << 33) return FISHING_ERR_SIZE;    // threads of a launch over the head, in 32 bits
    return FISHING_OK;
}

// the copies that are asked for, in one launch
template <typename T>
static int pads(const PadJob<T>& a, const PadJob<T>& b, const LossPlan& p, int64_t dim, int target_bytes, int64_t levels, hipStream_t stream) {
    auto blocks = [&](const PadJob<T>& j) { return j.src ? ceil_div(j.rows * (p.dim_p / vec_of<T>()), 256) : 0; };
    const int64_t first = blocks(a), second = blocks(b);
    if (first + second == 0) return 0;
    return launch(pad_kernel<T>, dim3((unsigned)(first + second)), dim3(256), stream, a, b, first, (int32_t)dim, (int32_t)p.dim_p, target_bytes, levels);
}

// the operand as it is where its rows are whole k steps at 16-byte addresses, its padded copy (whose job is then set) otherwise
template <typename T>
static Operand<T> padded_operand(const LossPlan& p, const T* src, int64_t ld, int64_t rows, int64_t dim, T* copy, PadJob<T>& job) {
    if (dim == p.dim_p && ld % vec_of<T>() == 0 && aligned16(src) && ld * (int64_t)sizeof(T) <= kMaxPitch) return Operand<T>{src, ld, rows, rows};
    job = PadJob<T>{src, ld, rows, copy, nullptr};
    return Operand<T>{copy, p.dim_p, rows, rows};
}

template <typename T>
static int loss_forward(int64_t rows, int64_t levels, int64_t dim, const T* h, int64_t h_ld, const T* w, int64_t w_ld, const void* target, int target_bytes, float* loss,
                        float* lse, void* workspace, hipStream_t stream) {
    const LossPlan p = loss_plan<T>(rows, levels, dim, false);
    const LossWork<T> k = loss_work<T>(p, rows, levels, dim, false, workspace);
    PadJob<T> w_job{};
    const Operand<T> b = padded_operand<T>(p, w, w_ld, levels, dim, k.w, w_job);
    int rc = 0;
    for (int64_t r0 = 0; r0 < rows && !rc; r0 += p.block) {
        const int64_t here = rows - r0 < p.block ? rows - r0 : p.block;
        const void* y = (const char*)target + r0 * target_bytes;
        PadJob<T> h_job{};
        const Operand<T> a = padded_operand<T>(p, h + r0 * h_ld, h_ld, here, dim, k.h, h_job);
        rc = pads(h_job, r0 ? PadJob<T>{} : w_job, p, dim, target_bytes, levels, stream);
        if (rc) break;
        rc = with_tile<T, false, false>(p.z, [&](auto t) {
            typedef decltype(t) Tile;
            const int64_t tm = ceil_div(here, Tile::EDGE), tn = ceil_div(levels, Tile::EDGE);
            return launch(loss_part_kernel<T, typename Tile::G, Tile::EDGE, Tile::EDGE>, dim3((unsigned)(tm * tn)), dim3(Tile::G::THREADS), stream, a, b, p.dim_p, y, target_bytes,
                          tm, tn, k.top, k.sum, k.taken);
        });
        if (rc) break;
        auto join_parts = [&](auto kernel, int r, int l) {
            return launch(kernel, dim3((unsigned)ceil_div(here, r)), dim3(r * l), stream, k.top, k.sum, k.taken, y, target_bytes, here, levels, p.parts, loss + r0, lse + r0);
        };
        rc = p.parts <= 8 ? join_parts(loss_join_kernel<256, 1>, 256, 1) : p.parts <= 64 ? join_parts(loss_join_kernel<32, 8>, 32, 8)
             : here <= 4096 ? join_parts(loss_join_kernel<4, 256>, 4, 256) : join_parts(loss_join_kernel<32, 32>, 32, 32);
    }
    return rc;
}

template <typename T, typename O, bool A_MAJOR, bool B_MAJOR, bool PADDED>
static int product(const Operand<T>& a, const Operand<T>& b, const Tiling& t, int64_t k, int64_t m, int64_t n, bool add, O* out, int64_t ld, int64_t slab, const Targets& y,
                   hipStream_t stream) {
    return with_tile<T, A_MAJOR, B_MAJOR>(t.b, [&](auto tile) {
        typedef decltype(tile) Tile;
        const int64_t tm = ceil_div(m, Tile::EDGE), tn = ceil_div(n, Tile::EDGE);
        return launch(product_kernel<T, O, typename Tile::G, Tile::EDGE, Tile::EDGE, PADDED>, dim3((unsigned)(tm * tn), (unsigned)t.shares), dim3(Tile::G::THREADS), stream, a, b, k,
                      t.share, m, n, tm, tn, add, out, ld, slab, y);
    });
}

template <typename T>
static int loss_backward(int64_t rows, int64_t levels, int64_t dim, const T* h, int64_t h_ld, const T* w, int64_t w_ld, const void* target, int target_bytes, const float* lse,
                         const float* g, T* dh, T* dw, void* workspace, hipStream_t stream) {
    const LossPlan p = loss_plan<T>(rows, levels, dim, true);
    const LossWork<T> k = loss_work<T>(p, rows, levels, dim, true, workspace);
    const Tiling whole = dw_tiling<T>(p, p.piece, dim);
    PadJob<T> w_job{};
    const Operand<T> b = padded_operand<T>(p, w, w_ld, levels, dim, k.w, w_job);
    int rc = 0;
    for (int64_t r0 = 0; r0 < rows && !rc; r0 += p.block) {
        const int64_t here = rows - r0 < p.block ? rows - r0 : p.block, here_p = round_up(here, p.bk);
        const void* y = (const char*)target + r0 * target_bytes;
        const Targets targets{y, target_bytes, levels};
        const Operand<T> a{k.h, p.dim_p, here, here};
        rc = pads(PadJob<T>{h + r0 * h_ld, h_ld, here, k.h, y}, r0 ? PadJob<T>{} : w_job, p, dim, target_bytes, levels, stream);
        for (int64_t v0 = 0; v0 < levels && !rc; v0 += p.piece) {
            const int64_t width = levels - v0 < p.piece ? levels - v0 : p.piece, width_p = round_up(width, p.bk);
            rc = with_tile<T, false, false>(tiling<T>(here, width, dim, false).b, [&](auto t) {
                typedef decltype(t) Tile;
                const int64_t tm = ceil_div(here, Tile::EDGE), tn = ceil_div(width, Tile::EDGE);
                return launch(loss_dz_kernel<T, typename Tile::G, Tile::EDGE, Tile::EDGE>, dim3((unsigned)(tm * tn)), dim3(Tile::G::THREADS), stream, a, b, p.dim_p, y, target_bytes,
                              levels, v0, tm, tn, lse + r0, g + r0, k.dzt, here_p);
            });
            if (rc) break;
            // dh[r][d]: m = d, n = r, k = the piece's levels, both operands k-major; W's rows beyond the last meet zeros of dz
            const Operand<T> wd{b.p + v0 * b.ld, b.ld, p.dim_p, width}, zr{k.dzt, here_p, here_p, width_p};
            Tiling t = width == p.piece ? p.dh : tiling<T>(dim, here, width, true);
            if (t.shares > p.dh.shares) {                       // (the first piece's slabs are all there are)
                t.share = round_up(ceil_div(width_p, p.dh.shares), p.bk);
                t.shares = ceil_div(width_p, t.share);
            }
            rc = k.dh ? product<T, float, true, true, true>(wd, zr, t, width_p, dim, here, v0 > 0, k.dh, dim, k.dh_slab, targets, stream)
                      : product<T, T, true, true, true>(wd, zr, t, width_p, dim, here, false, dh + r0 * dim, dim, 0, targets, stream);
            if (rc) break;
            // dW[v][d]: m = d, n = v, k = rows; h's rows beyond the last meet zeros of dz.  (A share behind the last block's rows adds
            // nothing to its slab.)
            const Operand<T> hd{k.h, p.dim_p, p.dim_p, here}, zv{k.dzt, here_p, width, width};
            t = k.dw_slab ? whole : dw_tiling<T>(p, width, dim);
            if (k.dw_slab) {
                rc = product<T, float, true, false, false>(hd, zv, t, here_p, dim, width, r0 > 0, k.dw + v0 * dim, dim, k.dw_slab, targets, stream);
            } else if (t.shares > 1) {
                const int64_t slab = round_up(width * dim, 4);
                rc = product<T, float, true, false, false>(hd, zv, t, here_p, dim, width, false, k.dw, dim, slab, targets, stream);
                if (!rc) rc = slab_sum<T>(k.dw, slab, t.shares, dw + v0 * dim, width * dim, stream);
            } else {
                rc = product<T, T, true, false, false>(hd, zv, t, here_p, dim, width, false, dw + v0 * dim, dim, 0, targets, stream);
            }
        }
        if (!rc && k.dh) rc = slab_sum<T>(k.dh, k.dh_slab, p.dh.shares, dh + r0 * dim, here * dim, stream);
    }
    if (!rc && k.dw_slab) rc = slab_sum<T>(k.dw, k.dw_slab, whole.shares, dw, levels * dim, stream);
    return rc;
}

}  // namespace seq
}  // namespace fishing

using namespace fishing::seq;

extern "C" {

int64_t fishing_cross_entropy_workspace(int32_t dtype, int64_t rows, int64_t levels, int64_t dim, int32_t backward) {
    if (int rc = loss_check(dtype, rows, levels, dim)) return rc;
    return dtype == FISHING_DTYPE_F32 ? loss_work<float>(loss_plan<float>(rows, levels, dim, backward != 0), rows, levels, dim, backward != 0, nullptr).bytes
                                      : loss_work<bf16>(loss_plan<bf16>(rows, levels, dim, backward != 0), rows, levels, dim, backward != 0, nullptr).bytes;
}

int fishing_cross_entropy_forward(int32_t dtype, int32_t target_bytes, int64_t rows, int64_t levels, int64_t dim, const void* hidden, int64_t hidden_stride, const void* head,
                                  int64_t head_stride, const void* target, float* loss, float* lse, void* workspace, int64_t workspace_bytes, fishing_stream_t stream) {
    if (int rc = loss_check(dtype, rows, levels, dim)) return rc;
    if (target_bytes != 4 && target_bytes != 8) return FISHING_ERR_UNSUPPORTED;
    if (hidden_stride < dim || head_stride < dim) return FISHING_ERR_SIZE;
    if (rows == 0) return FISHING_OK;
    if (!hidden || !head || !target || !loss || !lse || !workspace) return FISHING_ERR_NULL;
    if (!aligned16(workspace)) return FISHING_ERR_ALIGN;
    if (workspace_bytes < fishing_cross_entropy_workspace(dtype, rows, levels, dim, 0)) return FISHING_ERR_SIZE;
    hipStream_t st = (hipStream_t)stream;
    return dtype == FISHING_DTYPE_F32
               ? loss_forward<float>(rows, levels, dim, (const float*)hidden, hidden_stride, (const float*)head, head_stride, target, target_bytes, loss, lse, workspace, st)
               : loss_forward<bf16>(rows, levels, dim, (const bf16*)hidden, hidden_stride, (const bf16*)head, head_stride, target, target_bytes, loss, lse, workspace, st);
}

int fishing_cross_entropy_backward(int32_t dtype, int32_t target_bytes, int64_t rows, int64_t levels, int64_t dim, const void* hidden, int64_t hidden_stride, const void* head,
                                   int64_t head_stride, const void* target, const float* lse, const float* grad, void* dhidden, void* dhead, void* workspace,
                                   int64_t workspace_bytes, fishing_stream_t stream) {
    if (int rc = loss_check(dtype, rows, levels, dim)) return rc;
    if (target_bytes != 4 && target_bytes != 8) return FISHING_ERR_UNSUPPORTED;
    if (hidden_stride < dim || head_stride < dim) return FISHING_ERR_SIZE;
    if (!head || !dhead || !workspace || (rows > 0 && (!hidden || !target || !lse || !grad || !dhidden))) return FISHING_ERR_NULL;
    if (!aligned16(workspace)) return FISHING_ERR_ALIGN;
    if (workspace_bytes < fishing_cross_entropy_workspace(dtype, rows, levels, dim, 1)) return FISHING_ERR_SIZE;
    hipStream_t st = (hipStream_t)stream;
    if (rows == 0) {
        const int64_t blocks = ceil_div(levels * dim, 256);
        const dim3 grid((unsigned)(blocks < 65536 ? blocks : 65536));
        return dtype == FISHING_DTYPE_F32 ? launch(zero_kernel<float>, grid, dim3(256), st, (float*)dhead, levels * dim)
                                          : launch(zero_kernel<bf16>, grid, dim3(256), st, (bf16*)dhead, levels * dim);
    }
    return dtype == FISHING_DTYPE_F32 ? loss_backward<float>(rows, levels, dim, (const float*)hidden, hidden_stride, (const float*)head, head_stride, target, target_bytes, lse,
                                                             grad, (float*)dhidden, (float*)dhead, workspace, st)
                                      : loss_backward<bf16>(rows, levels, dim, (const bf16*)hidden, hidden_stride, (const bf16*)head, head_stride, target, target_bytes, lse,
                                                            grad, (bf16*)dhidden, (bf16*)dhead, workspace, st);
}

}  // extern "C"
