// sequence_loss.hip -- softmax cross entropy over the quota levels, in pieces of the levels, without keeping the logits.
//
//   z = h W^T        lse = log sum_v exp(z_v)        loss = lse - z_y        (0 where the target y is outside [0, levels))
//   dz = g (exp(z - lse) - [v == y])        dh = dz W        dW = dz^T h
//
// Forward: a workgroup computes the logits of a tile of rows against a range of levels and keeps each row's running maximum and sum;
// the ranges' pairs are joined afterwards.  Backward: the logits are computed again, a piece of the levels at a time, turned into dz
// in the operands' type (the factor of the two products' operands; sums stay in float32) and multiplied.
#include "sequence_common.h"

namespace fishing {
namespace seq {

// ---- a 64 x 64 tile of A B^T or its transposed forms; element (row, k) of an operand sits at row * ld + k, or k * ld + row ----
template <typename T>
struct Operand {
    const T* p;
    int64_t ld;
    int64_t rows;
    bool across;
    const void* target = nullptr;   // where given: k runs over rows of `hidden`, and those of padded targets count as zeros, whatever they hold
    int target_bytes = 0;
    int64_t levels = 0;
};

__device__ __forceinline__ int64_t target_of(const void* target, int bytes, int64_t row) {
    return bytes == 4 ? (int64_t)((const int32_t*)target)[row] : ((const int64_t*)target)[row];
}

template <typename T>
struct Tile {
    static constexpr int BK = 32, PAD = 8;
    T a[64][BK + PAD], b[64][BK + PAD];
};

template <typename T>
__device__ __forceinline__ void stage(T (*to)[Tile<T>::BK + Tile<T>::PAD], const Operand<T>& o, int64_t row0, int64_t k0, int64_t depth) {
    constexpr int BK = Tile<T>::BK;
    for (int x = threadIdx.x; x < 64 * BK; x += 256) {
        const int r = o.across ? x % 64 : x / BK, k = o.across ? x / 64 : x % BK;
        const int64_t row = row0 + r, kk = k0 + k;
        T e = from_f32<T>(0.0f);
        bool there = row < o.rows && kk < depth;
        if (there && o.target) {
            const int64_t y = target_of(o.target, o.target_bytes, kk);
            there = y >= 0 && y < o.levels;
        }
        if (there) e = o.across ? o.p[kk * o.ld + row] : o.p[row * o.ld + kk];
        to[r][k] = e;
    }
}

// four waves, each 32 x 32 as 2 x 2 matrix-core tiles
template <typename T>
__device__ __forceinline__ void multiply(Tile<T>& t, const Operand<T>& a, int64_t a0, const Operand<T>& b, int64_t b0, int64_t depth, f32x4 (&acc)[2][2]) {
    typedef Mma<T> M;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, wr = (wave >> 1) * 32, wc = (wave & 1) * 32;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int64_t k0 = 0; k0 < depth; k0 += Tile<T>::BK) {
        __syncthreads();
        stage<T>(t.a, a, a0, k0, depth);
        stage<T>(t.b, b, b0, k0, depth);
        __syncthreads();
#pragma unroll
        for (int k = 0; k < Tile<T>::BK; k += M::K) {
            typename M::Frag fa[2], fb[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                fa[i] = *(const typename M::Frag*)&t.a[wr + i * 16 + lane % 16][k + (lane / 16) * M::E];
                fb[i] = *(const typename M::Frag*)&t.b[wc + i * 16 + lane % 16][k + (lane / 16) * M::E];
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[i][j] = M::run(fa[i], fb[j], acc[i][j]);
        }
    }
}

template <typename F>
__device__ __forceinline__ void each(f32x4 (&acc)[2][2], F f) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, wr = (wave >> 1) * 32, wc = (wave & 1) * 32;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) f(wr + i * 16 + (lane / 16) * 4 + r, wc + j * 16 + lane % 16, acc[i][j][r]);
}


template <typename T>
__global__ void __launch_bounds__(256) loss_part_kernel(Operand<T> h, Operand<T> w, int64_t dim, const void* target, int target_bytes, int64_t span, float* top, float* sum,
                                                        float* taken) {
    __shared__ Tile<T> t;
    __shared__ float z[64][65];
    const int64_t r0 = (int64_t)blockIdx.x * 64, lo = blockIdx.y * span, hi = lo + span < w.rows ? lo + span : w.rows;
    float m = -INFINITY, s = 0.0f;          // thread r < 64 keeps row r's
    for (int64_t v0 = lo; v0 < hi; v0 += 64) {
        f32x4 acc[2][2];
        multiply<T>(t, h, r0, w, v0, dim, acc);
        each(acc, [&](int r, int c, float x) { z[r][c] = x; });
        __syncthreads();
        const int64_t row = r0 + threadIdx.x;
        if (threadIdx.x < 64 && row < h.rows) {
            const int n = hi - v0 < 64 ? (int)(hi - v0) : 64;
            float now = m;
            for (int c = 0; c < n; ++c) now = z[threadIdx.x][c] > now || z[threadIdx.x][c] != z[threadIdx.x][c] ? z[threadIdx.x][c] : now;
            s = m == now ? s : s * expf(m - now);
            for (int c = 0; c < n; ++c) s += z[threadIdx.x][c] == now && fabsf(now) == INFINITY ? 1.0f : expf(z[threadIdx.x][c] - now);
            m = now;
            const int64_t y = target_of(target, target_bytes, row);
            if (y >= v0 && y < v0 + n) taken[row] = z[threadIdx.x][y - v0];
        }
    }
    const int64_t row = r0 + threadIdx.x;
    if (threadIdx.x < 64 && row < h.rows) {
        top[blockIdx.y * h.rows + row] = m;
        sum[blockIdx.y * h.rows + row] = s;
    }
}

__global__ void __launch_bounds__(256) loss_join_kernel(const float* top, const float* sum, const float* taken, const void* target, int target_bytes, int64_t rows,
                                                        int64_t levels, int parts, float* loss, float* lse) {
    const int64_t row = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (row >= rows) return;
    float m = -INFINITY;
    for (int p = 0; p < parts; ++p) {
        const float x = top[p * rows + row];
        m = x > m || x != x ? x : m;
    }
    float s = 0.0f;
    for (int p = 0; p < parts; ++p) s += top[p * rows + row] == m ? sum[p * rows + row] : sum[p * rows + row] * expf(top[p * rows + row] - m);
    const float l = m + logf(s);
    lse[row] = l;
    const int64_t y = target_of(target, target_bytes, row);
    loss[row] = y >= 0 && y < levels ? l - taken[row] : 0.0f;
}

// a piece of dz: rows x [v0, v0 + width)
template <typename T>
__global__ void __launch_bounds__(256) loss_dz_kernel(Operand<T> h, Operand<T> w, int64_t dim, const void* target, int target_bytes, int64_t levels, int64_t v0,
                                                      int64_t width, const float* lse, const float* g, T* dz) {
    __shared__ Tile<T> t;
    f32x4 acc[2][2];
    const int64_t r0 = (int64_t)blockIdx.x * 64, c0 = (int64_t)blockIdx.y * 64;
    multiply<T>(t, h, r0, w, v0 + c0, dim, acc);
    each(acc, [&](int r, int c, float x) {
        const int64_t row = r0 + r, col = c0 + c;
        if (row >= h.rows || col >= width) return;
        const int64_t y = target_of(target, target_bytes, row);
        const float p = expf(x - lse[row]) - (y == v0 + col ? 1.0f : 0.0f);
        dz[row * width + col] = from_f32<T>(y >= 0 && y < levels ? g[row] * p : 0.0f);
    });
}

// out (+)= A B^T over the depth; to float32 (kept between pieces) or to the type
template <typename T, typename O, bool ADD>
__global__ void __launch_bounds__(256) product_kernel(Operand<T> a, Operand<T> b, int64_t depth, const float* before, O* out, int64_t ld) {
    __shared__ Tile<T> t;
    f32x4 acc[2][2];
    const int64_t r0 = (int64_t)blockIdx.x * 64, c0 = (int64_t)blockIdx.y * 64;
    multiply<T>(t, a, r0, b, c0, depth, acc);
    each(acc, [&](int r, int c, float x) {
        const int64_t row = r0 + r, col = c0 + c;
        if (row >= a.rows || col >= b.rows) return;
        out[row * ld + col] = from_f32<O>(ADD ? before[row * ld + col] + x : x);
    });
}

struct LossPlan {
    int64_t span, piece;
    int parts;
};

static LossPlan loss_plan(int64_t rows, int64_t levels) {
    LossPlan p;
    const int64_t want = ceil_div(2048, ceil_div(rows > 0 ? rows : 1, 64));
    p.span = round_up(ceil_div(levels, want), 64);
    p.parts = (int)ceil_div(levels, p.span);
    p.piece = levels < 16384 ? levels : 16384;
    return p;
}

struct LossWork {
    float *top, *sum, *taken, *dh;
    void* dz;
    int64_t bytes;
};

static LossWork loss_work(const LossPlan& p, int64_t size, int64_t rows, int64_t levels, int64_t dim, bool backward, void* at) {
    Carve c(at);
    LossWork w{};
    if (backward) {
        w.dz = c.take<char>(rows * p.piece * size);
        w.dh = c.take<float>(p.piece < levels ? rows * dim : 0);
    } else {
        w.top = c.take<float>(rows * p.parts);
        w.sum = c.take<float>(rows * p.parts);
        w.taken = c.take<float>(rows);
    }
    w.bytes = c.used + 256;
    return w;
}

static int loss_check(int32_t dtype, int64_t rows, int64_t levels, int64_t dim) {
    if (dtype != FISHING_DTYPE_F32 && dtype != FISHING_DTYPE_BF16) return FISHING_ERR_UNSUPPORTED;
    if (rows < 0 || rows > 0x7fffffff || levels < 1 || levels > 0x7ffffff || dim < 1 || dim > 65536) return FISHING_ERR_SIZE;
    return FISHING_OK;
}

template <typename T>
static int loss_forward(int64_t rows, int64_t levels, int64_t dim, const T* h, int64_t h_ld, const T* w, int64_t w_ld, const void* target, int target_bytes, float* loss,
                        float* lse, void* workspace, hipStream_t stream) {
    const LossPlan p = loss_plan(rows, levels);
    const LossWork k = loss_work(p, sizeof(T), rows, levels, dim, false, workspace);
    const Operand<T> a{h, h_ld, rows, false}, b{w, w_ld, levels, false};
    int rc = launch(loss_part_kernel<T>, dim3((unsigned)ceil_div(rows, 64), (unsigned)p.parts), dim3(256), stream, a, b, dim, target, target_bytes, p.span, k.top, k.sum, k.taken);
    if (!rc)
        rc = launch(loss_join_kernel, dim3((unsigned)ceil_div(rows, 256)), dim3(256), stream, k.top, k.sum, k.taken, target, target_bytes, rows, levels, p.parts, loss, lse);
    return rc;
}

template <typename T>
static int loss_backward(int64_t rows, int64_t levels, int64_t dim, const T* h, int64_t h_ld, const T* w, int64_t w_ld, const void* target, int target_bytes, const float* lse,
                         const float* g, T* dh, T* dw, void* workspace, hipStream_t stream) {
    const LossPlan p = loss_plan(rows, levels);
    const LossWork k = loss_work(p, sizeof(T), rows, levels, dim, true, workspace);
    T* dz = (T*)k.dz;
    const Operand<T> a{h, h_ld, rows, false};
    int rc = 0;
    for (int64_t v0 = 0; v0 < levels && !rc; v0 += p.piece) {
        const int64_t width = levels - v0 < p.piece ? levels - v0 : p.piece;
        const bool first = v0 == 0, last = v0 + width == levels;
        const Operand<T> all{w, w_ld, levels, false}, rowwise{dz, width, rows, false}, levelwise{dz, width, width, true};
        const Operand<T> w_dim{w + v0 * w_ld, w_ld, dim, true}, h_dim{h, h_ld, dim, true, target, target_bytes, levels};
        rc = launch(loss_dz_kernel<T>, dim3((unsigned)ceil_div(rows, 64), (unsigned)ceil_div(width, 64)), dim3(256), stream, a, all, dim, target, target_bytes, levels, v0, width,
                    lse, g, dz);
        const dim3 grid((unsigned)ceil_div(rows, 64), (unsigned)ceil_div(dim, 64));
        if (!rc) {
            if (first && last)
                rc = launch(product_kernel<T, T, false>, grid, dim3(256), stream, rowwise, w_dim, width, k.dh, dh, dim);
            else if (first)
                rc = launch(product_kernel<T, float, false>, grid, dim3(256), stream, rowwise, w_dim, width, k.dh, k.dh, dim);
            else if (!last)
                rc = launch(product_kernel<T, float, true>, grid, dim3(256), stream, rowwise, w_dim, width, k.dh, k.dh, dim);
            else
                rc = launch(product_kernel<T, T, true>, grid, dim3(256), stream, rowwise, w_dim, width, k.dh, dh, dim);
        }
        if (!rc)
            rc = launch(product_kernel<T, T, false>, dim3((unsigned)ceil_div(width, 64), (unsigned)ceil_div(dim, 64)), dim3(256), stream, levelwise, h_dim, rows, k.dh,
                        dw + v0 * dim, dim);
    }
    return rc;
}

template <typename T>
__global__ void __launch_bounds__(256) zero_kernel(T* p, int64_t n) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < n) p[i] = from_f32<T>(0.0f);
}

}  // namespace seq
}  // namespace fishing

using namespace fishing::seq;

extern "C" {

int64_t fishing_cross_entropy_workspace(int32_t dtype, int64_t rows, int64_t levels, int64_t dim, int32_t backward) {
    if (int rc = loss_check(dtype, rows, levels, dim)) return rc;
    return loss_work(loss_plan(rows, levels), dtype == FISHING_DTYPE_F32 ? 4 : 2, rows, levels, dim, backward != 0, nullptr).bytes;
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
        const dim3 grid((unsigned)ceil_div(levels * dim, 256));
        return dtype == FISHING_DTYPE_F32 ? launch(zero_kernel<float>, grid, dim3(256), st, (float*)dhead, levels * dim)
                                          : launch(zero_kernel<bf16>, grid, dim3(256), st, (bf16*)dhead, levels * dim);
    }
    return dtype == FISHING_DTYPE_F32 ? loss_backward<float>(rows, levels, dim, (const float*)hidden, hidden_stride, (const float*)head, head_stride, target, target_bytes, lse,
                                                             grad, (float*)dhidden, (float*)dhead, workspace, st)
                                      : loss_backward<bf16>(rows, levels, dim, (const bf16*)hidden, hidden_stride, (const bf16*)head, head_stride, target, target_bytes, lse,
                                                            grad, (bf16*)dhidden, (bf16*)dhead, workspace, st);
}

}  // extern "C"
