// sequence_walk.h -- linear attention's walk over whole episodes: the chunk kernels, what repairs values that are not numbers, and the
// walk's plan and launches.  Instantiated forwards in sequence_attention.hip and backwards in sequence_attention_back.hip.
#pragma once
#include "sequence_common.h"

namespace fishing {
namespace seq {

constexpr int kMaxHeadDim = 128;

struct Strided {
    const void* p;
    int64_t batch, step, head;
};

// exp(-inf * 0) would be NaN: a decay of zero is carried as a logarithm far below float32's range (and NaN stays NaN)
__device__ __forceinline__ float log_decay_of(const float* log_decay, int h) { return log_decay[h] < -1.0e4f ? -1.0e4f : log_decay[h]; }

// Batches are walked in blocks whose launches' threads count in 32 bits: 2^22 (batch, head) pairs, four 64-lane waves each at most
constexpr int kMaxHeads = 65536;
static int64_t batch_block(int64_t batch, int heads) {
    const int64_t most = ((int64_t)1 << 22) / heads;
    return batch < most ? batch : most;
}

// ---- whole episodes, a chunk of 32 (f32: 16) steps at a time: one wave owns a (batch, head), up to 64 columns of its state, and a run of steps ----
//
// With g = exp(log_decay) and the steps x of a chunk of n, "open" meaning that no start lies between:
//   forwards   o_x = sum_{y <= x, open} g^(x-y) (q_x . k_y) v_y + [open to the chunk's front] g^(x+1) q_x S
//              S' = [no start] g^n S + sum_{y, open to the end} g^(n-1-y) k_y v_y^T
//   backwards  o_x = sum_{y >= x, open} g^(y-x) (q_x . k_y) v_y + [open to the chunk's end] g^(n-1-x) q_x S
//              S' = [no start] g^n S + sum_{y, no start in 0 .. y} g^(y+1) k_y v_y^T
// so a chunk is four small products on the matrix cores.  The layouts chain without a shuffle: the tile k q^T has its columns in
// lanes and four rows y in registers, which is the second operand of v^T (k q^T); a state tile k^T v likewise is the first of S^T q^T;
// the outputs come as four neighbouring columns of one step per lane.  k and v are read by columns through the transposing LDS read
// (bf16) or element reads (f32).  bf16: the products need scores, the state and the decayed v in bf16.  The state's copy and the scores
// go as two bf16 terms (16 bits) and the decayed v as two or, where the state is an answer in float32, three: what comes before an
// output's own rounding is then too small to show in it (a copy of the state in one term: up to 1.4x that rounding, 2 - 3% less time).
// A wave alone needs no barriers; the next chunk's rows are loaded into registers while this one is computed, and the registers (state,
// rows in flight, operands) leave room for two waves on a SIMD.  What bounds it is those waves' dependent work, not a unit: 2048 x 101
// steps, 4 heads of 64 x 64, bf16: 117 us a walk, 3.6 TB/s of operands, VALU 42% and matrix cores 18% busy; 97 x 1009 steps, 3 heads of
// 48 x 80, f32: 76 - 98 us and 44 for the segments' states, matrix cores 44% busy; 16381 steps, 8 heads of 128 x 128, bf16, one wave a
// SIMD: 67 us, states 27, chain 11.  (A third wave a SIMD spilled: 2.3 times slower.)  Rows that are not whole 16-byte accesses take
// element loads, and two tiles of columns a wave: 2048 x 101 steps of 63 x 65 instead of 64 x 64 with gradients 2092 us for 479, 97 x 1009 of
// 47 x 81 f32 1074 for 509 (kernels, captured).

// The value, not to be worked with ahead of this place: what is computed of lane numbers for the rare chunk would otherwise be
// computed once and kept, some sixty registers of it
__device__ __forceinline__ int here(int x) {
    asm volatile("" : "+v"(x));
    return x;
}
__device__ __forceinline__ uint32_t here(uint32_t x) { return (uint32_t)here((int)x); }

template <typename T>
struct Lanes;
template <>
struct Lanes<bf16> {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef s16x4 Quad;
    static constexpr bool SPLIT = true;
    static constexpr int TILES = 2;            // of 16 steps in a chunk: the products over steps take 32 at once
    // four steps y of one column; each lane names the 8 bytes (4 columns of one step) that it contributes
    static __device__ __forceinline__ Quad column(const char* rows, int pitch, int y0, int col, int spread) {
        const int i = threadIdx.x & 15, g = threadIdx.x >> 4 & 3;
        const char* at = rows + (y0 + 4 * g + (i >> 2)) * pitch + (col + spread * (i & 3)) * 2;
        return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)at);
    }
    static __device__ __forceinline__ Quad state_column(const char* rows, int pitch, int y0, int c) { return column(rows, pitch, y0, 32 * (c >> 1) + 4 * (c & 1), 8); }
    static __device__ __forceinline__ Quad value_column(const char* rows, int pitch, int y0, int n) { return column(rows, pitch, y0, 16 * n, 4); }
    // eight neighbouring elements of one row, as the quads of tiles 2c and 2c + 1
    static __device__ __forceinline__ void row_quads(const char* rows, int pitch, int y, int c, Quad& a, Quad& b) {
        const int g = threadIdx.x >> 4 & 3;
        typedef short s16x8 __attribute__((ext_vector_type(8)));
        const s16x8 x = *(const s16x8*)(rows + y * pitch + (32 * c + 8 * g) * 2);
        a = __builtin_shufflevector(x, x, 0, 1, 2, 3);
        b = __builtin_shufflevector(x, x, 4, 5, 6, 7);
    }
    // the state tile c's row 4 g + r
    static __device__ __forceinline__ int state_row(int c, int g) { return 32 * (c >> 1) + 8 * g + 4 * (c & 1); }
    // of row x: its tile, and its place in a tile's 16 (4 g + r)
    static __device__ __forceinline__ int row_tile(int x) { return 2 * (x >> 5) + (x >> 2 & 1); }
    static __device__ __forceinline__ int row_place(int x) { return 4 * (x >> 3 & 3) + (x & 3); }
    static __device__ __forceinline__ f32x4 mma(Quad a0, Quad a1, Quad b0, Quad b1, f32x4 acc) {
        union {
            Quad q[2];
            bf16x8 f;
        } a{{a0, a1}}, b{{b0, b1}};
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.f, b.f, acc, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x4 over_steps(const Quad (&a)[2], const Quad (&b)[2], f32x4 acc) { return mma(a[0], a[1], b[0], b[1], acc); }
    // (two at a time, v_cvt_pk_bf16_f32; element by element the halves would live in registers of their own)
    static __device__ __forceinline__ Quad round(f32x4 x) {
        union {
            bf16x4 h;
            Quad q;
        } y;
        y.h = __builtin_convertvector(x, bf16x4);
        return y.q;
    }
    static __device__ __forceinline__ f32x4 wide(Quad x) {
        union {
            Quad q;
            uint32_t u[2];
        } y{x};
        return f32x4{__uint_as_float(y.u[0] << 16), __uint_as_float(y.u[0] & 0xffff0000u), __uint_as_float(y.u[1] << 16), __uint_as_float(y.u[1] & 0xffff0000u)};
    }
};
template <>
struct Lanes<float> {
    typedef f32x4 Quad;
    static constexpr bool SPLIT = false;
    static constexpr int TILES = 1;            // the products over steps take 4 at once: longer chunks would only add masked scores
    static __device__ __forceinline__ Quad column(const char* rows, int pitch, int y0, int col) {
        const int i = threadIdx.x & 15, g = threadIdx.x >> 4 & 3;
        Quad x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = *(const float*)(rows + (y0 + 4 * g + e) * pitch + (col + i) * 4);
        return x;
    }
    static __device__ __forceinline__ Quad state_column(const char* rows, int pitch, int y0, int c) { return column(rows, pitch, y0, 16 * c); }
    static __device__ __forceinline__ Quad value_column(const char* rows, int pitch, int y0, int n) { return column(rows, pitch, y0, 16 * n); }
    static __device__ __forceinline__ void row_quads(const char* rows, int pitch, int y, int c, Quad& a, Quad& b) {
        const int g = threadIdx.x >> 4 & 3;
        a = *(const Quad*)(rows + y * pitch + (32 * c + 4 * g) * 4);
        b = *(const Quad*)(rows + y * pitch + (32 * c + 16 + 4 * g) * 4);
    }
    static __device__ __forceinline__ Quad row_quad(const char* rows, int pitch, int y, int c) { return *(const Quad*)(rows + y * pitch + (16 * c + 4 * (threadIdx.x >> 4 & 3)) * 4); }
    static __device__ __forceinline__ int state_row(int c, int g) { return 16 * c + 4 * g; }
    static __device__ __forceinline__ int row_tile(int x) { return x >> 4; }
    static __device__ __forceinline__ int row_place(int x) { return x & 15; }
    static __device__ __forceinline__ f32x4 mma(Quad a0, Quad a1, Quad b0, Quad b1, f32x4 acc) {
#pragma unroll
        for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a0[e], b0[e], acc, 0, 0, 0);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a1[e], b1[e], acc, 0, 0, 0);
        return acc;
    }
    static __device__ __forceinline__ f32x4 over_steps(const Quad (&a)[1], const Quad (&b)[1], f32x4 acc) {
#pragma unroll
        for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[0][e], b[0][e], acc, 0, 0, 0);
        return acc;
    }
    static __device__ __forceinline__ Quad round(f32x4 x) { return x; }
    static __device__ __forceinline__ f32x4 wide(Quad x) { return x; }
};

// A chunk's rows of one operand on their way from memory, 16 bytes a lane and load.  Rows behind the last and columns behind d are
// zeros.  VEC: buffer loads, which answer zeros for what lies behind the buffer: its length ends the rows, and a lane of columns
// behind d points there.  (Steps of at least d, 32 of them in 31 bits: the plan's business.)  No branch and no mask: with either the
// compiler could not count the loads and waited for one operand's before it sent the next's.
template <typename T, int TILES, int STEPS, bool VEC>
struct Rows {
    static constexpr int EPC = 16 / (int)sizeof(T), CHUNKS = TILES * 16 / EPC, LOADS = STEPS * CHUNKS / 64, PITCH = TILES * 16 * (int)sizeof(T) + 16;
    static constexpr bool EVEN = 64 % CHUNKS == 0;                    // (96 columns: 12 chunks a row do not divide the wave)
    static constexpr int PER = EVEN ? 64 / CHUNKS : 0;                // rows of a load
    static_assert(STEPS * CHUNKS % 64 == 0, "whole loads");
    u32x4 x[LOADS];

    static __device__ __forceinline__ int row_of(int s) { return EVEN ? (int)threadIdx.x / CHUNKS + s * PER : (s * 64 + (int)threadIdx.x) / CHUNKS; }
    static __device__ __forceinline__ int chunk_of(int s) { return EVEN ? (int)threadIdx.x % CHUNKS : (s * 64 + (int)threadIdx.x) % CHUNKS; }
    // a lane's place from a chunk's first row on
    static __device__ __forceinline__ uint32_t place(int s, int64_t step, int d) {
        const int c = chunk_of(s) * EPC;
        return c < d ? ((uint32_t)row_of(s) * (uint32_t)step + c) * (uint32_t)sizeof(T) : 0x80000000u;
    }
    uint32_t at[EVEN ? 1 : LOADS];
    __device__ __forceinline__ void init(int64_t step, int d) {
        if constexpr (VEC) {
#pragma unroll
            for (int s = 0; s < (EVEN ? 1 : LOADS); ++s) at[s] = place(s, step, d);
        }
    }
    // p: the chunk's first row (uniform)
    __device__ __forceinline__ void load(const T* p, int64_t step, int rows, int d) {
        if constexpr (VEC) {
            const auto buffer = __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, (uint32_t)((uint32_t)(rows - 1) * (uint32_t)step + d) * (uint32_t)sizeof(T), 0x00020000);
            const uint32_t next = (uint32_t)(PER * (int)sizeof(T)) * (uint32_t)step;
#pragma unroll
            for (int s = 0; s < LOADS; ++s) x[s] = __builtin_amdgcn_raw_buffer_load_b128(buffer, EVEN ? at[0] + s * next : at[EVEN ? 0 : s], 0, 0);
        } else {
#pragma unroll
            for (int s = 0; s < LOADS; ++s) {
                const int r = row_of(s), c = chunk_of(s) * EPC;
                const T* from = p + (r < rows ? r : rows - 1) * step;
                Pack<T, EPC> y;
#pragma unroll
                for (int e = 0; e < EPC; ++e) y.e[e] = r < rows && c + e < d ? from[c + e] : from_f32<T>(0.0f);
                x[s] = *(const u32x4*)&y;
            }
        }
    }
    __device__ __forceinline__ void put(char* lds) const {
        char* to = lds + threadIdx.x / CHUNKS * PITCH + threadIdx.x % CHUNKS * 16;
#pragma unroll
        for (int s = 0; s < LOADS; ++s) *(u32x4*)(EVEN ? to + s * PER * PITCH : lds + row_of(s) * PITCH + chunk_of(s) * 16) = x[s];
    }
};

struct ChunkArgs {
    Strided q, k, v, out;
    const float* log_decay;
    const uint8_t* starts;
    int64_t starts_batch, starts_step;
    const float* state;        // [batch, heads, dk, dv], or transposed: [batch, heads, dv, dk]
    float* state_out;
    int64_t steps;
    int32_t heads, dk, dv;
    bool state_t, exact_state;
    float read_scale, write_scale;
    int32_t slices, segs;
    int64_t seg_steps;
    float *carry, *through;    // the state behind a segment, per (pair, 16 columns, segment) in lane order, and what a segment lets through, per (pair, segment)
    uint32_t* odd;             // per (pair, slice, segment): some result is infinite or NaN
    int32_t carry_nk;          // not 0: the carry is that of a walk whose state is this one's transposed, this many tiles of rows
};

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
template <typename R>
__device__ __forceinline__ void store_quad(R rows, uint32_t at, int further, Lanes<bf16>::Quad x) {
    union {
        Lanes<bf16>::Quad q;
        u32x2 u;
    } y{x};
    __builtin_amdgcn_raw_buffer_store_b64(y.u, rows, at, further, 0);
}
template <typename R>
__device__ __forceinline__ void store_quad(R rows, uint32_t at, int further, f32x4 x) {
    union {
        f32x4 q;
        u32x4 u;
    } y{x};
    __builtin_amdgcn_raw_buffer_store_b128(y.u, rows, at, further, 0);
}

// Waves on a SIMD, by the registers that state, rows in flight and operands take: two where nothing spills, else one
constexpr int waves_a_simd(int nk, int nv, bool vec, bool local) {
    return local ? (nk * nv >= 24 ? 1 : 2) : nk * nv > 16 || nk == 8 || (!vec && nk >= 6) ? 1 : 2;
}

// LOCAL: only the state that a segment adds (from zero; the first from the state carried in), for the segments to be chained.
template <typename T, int NK, int NV, bool BACK, bool VEC, bool LOCAL>
__global__ void __launch_bounds__(64, waves_a_simd(NK, NV, VEC, LOCAL)) chunk_kernel(ChunkArgs a) {
    static_assert(sizeof(T) == 4 || NK % 2 == 0, "bf16 rows are multiplied 32 elements at a time");
    typedef Lanes<T> L;
    typedef typename L::Quad Quad;
    constexpr int TS = L::TILES, CH = 16 * TS;
    typedef Rows<T, NK, CH, VEC> RK;
    typedef Rows<T, NV, CH, VEC> RV;
    __shared__ __attribute__((aligned(16))) char qs[CH * RK::PITCH];
    __shared__ __attribute__((aligned(16))) char ks[CH * RK::PITCH];
    __shared__ __attribute__((aligned(16))) char vs[CH * RV::PITCH];
    const int lane = threadIdx.x, i = lane & 15, g = lane >> 4;
    // (slices of a pair read the same q and k: neighbours on one XCD)
    const uint32_t units = (uint32_t)(a.slices * a.segs);
    const int64_t id = xcd_run(blockIdx.x, gridDim.x), pair = uniform((int)((uint32_t)id / units));
    const int rest = (int)id - (int)pair * (int)units, slice = uniform((int)((uint32_t)rest / (uint32_t)a.segs)), seg = rest - slice * a.segs;
    if (LOCAL && seg == a.segs - 1) return;                  // nothing follows it
    const int64_t n = uniform((int)((uint32_t)pair / (uint32_t)a.heads)), h = pair - n * a.heads;
    const int col0 = slice * NV * 16, cols = a.dv - col0, col_tiles = (a.dv + 15) / 16;
    const T* qp = (const T*)a.q.p + n * a.q.batch + h * a.q.head;
    const T* kp = (const T*)a.k.p + n * a.k.batch + h * a.k.head;
    const T* vp = (const T*)a.v.p + n * a.v.batch + h * a.v.head + col0;
    T* op = (T*)a.out.p + n * a.out.batch + h * a.out.head + col0;
    // segments are counted in the direction of the walk
    const int64_t at = BACK ? a.segs - 1 - seg : seg, t_lo = at * a.seg_steps, t_hi = t_lo + a.seg_steps < a.steps ? t_lo + a.seg_steps : a.steps;
    const int chunks = (int)ceil_div(t_hi - t_lo, CH);
    const float ld = __int_as_float(uniform(__float_as_int(log_decay_of(a.log_decay, (int)h)))), l2 = ld * 1.4426950408889634f;
    const float whole = __int_as_float(uniform(__float_as_int((float)exp((double)ld * CH))));     // the factor that compounds: rounded once

    RK rq, rk;
    RV rv;
    rq.init(a.q.step, a.dk);
    rk.init(a.k.step, a.dk);
    rv.init(a.v.step, cols);
    const uint32_t starts_at = (uint32_t)lane * (uint32_t)a.starts_step;
    uint32_t started = 0;                         // the lane's step begins an episode (tested behind the wait for the rows)
    auto front = [&](int x) { return t_lo + (int64_t)(BACK ? chunks - 1 - x : x) * CH; };
    auto count = [&](int64_t t0) { return t_hi - t0 < CH ? (int)(t_hi - t0) : CH; };
    auto fetch = [&](int x) {
        const int64_t t0 = front(x);
        const int rows = count(t0);
        if (!LOCAL) rq.load(qp + t0 * a.q.step, a.q.step, rows, a.dk);
        rk.load(kp + t0 * a.k.step, a.k.step, rows, a.dk);
        rv.load(vp + t0 * a.v.step, a.v.step, rows, cols);
        if (a.starts) {
            const uint8_t* from = a.starts + n * a.starts_batch + t0 * a.starts_step;
            if constexpr (VEC)
                started = __builtin_amdgcn_raw_buffer_load_b8(__builtin_amdgcn_make_buffer_rsrc((void*)from, 0, (uint32_t)(rows - 1) * (uint32_t)a.starts_step + 1, 0x00020000),
                                                              starts_at, 0, 0);
            else
                started = from[(lane < rows ? lane : 0) * a.starts_step];
        }
    };
    if (chunks > 0) fetch(0);                     // (on their way while the weights are computed)

    // What a whole chunk without a start weighs its terms with, per lane: a score of steps d apart, in order, in tiles t apart; a step's
    // k v^T behind the chunk; the state in front of the chunk at a step.  In LDS: the registers are the rows' in flight.
    __shared__ f32x4 near_of[TS][64], behind_of[TS][64];
    __shared__ float ahead_of[TS][64];
#pragma unroll
    for (int t = 0; t < TS; ++t) {
        f32x4 x, y4;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int y = 4 * g + r, d = BACK ? y - i + 16 * t : i + 16 * t - y;
            x[r] = d >= 0 ? __builtin_amdgcn_exp2f(d * l2) * (a.read_scale * a.write_scale) : 0.0f;
            y4[r] = a.write_scale * __builtin_amdgcn_exp2f((BACK ? 16 * t + y + 1 : CH - 1 - (16 * t + y)) * l2);
        }
        near_of[t][lane] = x;
        behind_of[t][lane] = y4;
        ahead_of[t][lane] = a.read_scale * __builtin_amdgcn_exp2f((BACK ? CH - 1 - (16 * t + i) : 16 * t + i + 1) * l2);
    }

    f32x4 S[NK][NV];
    {
        const float* from = a.carry + ((pair * col_tiles + col0 / 16) * a.segs + seg - 1) * (NK * 256);
        const float* s0 = a.state ? a.state + pair * (int64_t)a.dk * a.dv : nullptr;
#pragma unroll
        for (int c = 0; c < NK; ++c)
#pragma unroll
            for (int m = 0; m < NV; ++m) {
                S[c][m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                if (BACK && !LOCAL && seg > 0 && a.carry_nk) {
                    const int col = col0 + m * 16 + i, row = L::state_row(c, g), tiles = (a.dk + 15) / 16;
                    const float* other = a.carry + ((pair * tiles + (row >> 4)) * a.segs + seg - 1) * (a.carry_nk * 256) + L::row_tile(col) * 256 + (L::row_place(col) >> 2) * 64 +
                                         (col & 3);
                    if (row < tiles * 16 && col < a.carry_nk * 16) {
#pragma unroll
                        for (int r = 0; r < 4; ++r) S[c][m][r] = other[((row & 15) + r) * 4];
                    }
                } else if (seg > 0) {
                    if (!LOCAL && col0 / 16 + m < col_tiles) S[c][m] = *(const f32x4*)(from + (m * a.segs * NK + c) * 256 + lane * 4);
                } else if (s0) {
                    const int col = m * 16 + i, row = L::state_row(c, g);
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (col < cols && row + r < a.dk) S[c][m][r] = a.state_t ? s0[(int64_t)(col0 + col) * a.dk + row + r] : s0[(int64_t)(row + r) * a.dv + col0 + col];
                }
            }
    }

    // S is kept as a multiple: the state is sigma * S.  A chunk's decay then costs one factor, not one per element (and none of the
    // moves between register files that those cost); past 2^-8 or 2^8, and where a start cuts, S is multiplied out.
    float odd = 0.0f, through = 1.0f, sigma = 1.0f;
    for (int x = 0; x < chunks; ++x) {
        const int64_t t0 = front(x);
        const int rows = count(t0);
        __syncthreads();
        if (!LOCAL) rq.put(qs);
        rk.put(ks);
        rv.put(vs);
        const uint32_t st = (uint32_t)__ballot(started != 0 && lane < rows);
        __syncthreads();
        f32x4 w[TS];
        float into[TS], pass = whole;
#pragma unroll
        for (int t = 0; t < TS; ++t) {
            w[t] = behind_of[t][lane];
            into[t] = ahead_of[t][lane];
        }
        if (st || rows != CH) {                   // uniform: few chunks
            const int g4 = here(4 * g), i0 = here(i);
            pass = st ? 0.0f : exp2f(rows * l2);
            const int from = !BACK && st ? 31 - __clz(st) : 0, to = BACK && st ? __ffs(st) - 1 : rows;
#pragma unroll
            for (int t = 0; t < TS; ++t) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int y = 16 * t + g4 + r;
                    w[t][r] = y >= from && y < to ? a.write_scale * __builtin_amdgcn_exp2f((BACK ? y + 1 : rows - 1 - y) * l2) : 0.0f;
                }
                const int step = 16 * t + i0;
                const uint32_t upto = (2u << step) - 1u, cuts = BACK ? st & ~upto : st & upto;
                into[t] = cuts || step >= rows ? 0.0f : a.read_scale * __builtin_amdgcn_exp2f((BACK ? rows - 1 - step : step + 1) * l2);
            }
        }
        through = st ? 0.0f : through * pass;
        const float decayed = __int_as_float(uniform(__float_as_int(sigma * pass)));
        const bool kept = decayed >= 0x1p-8f && decayed <= 0x1p8f;
        const float scale = kept ? 1.0f / decayed : 1.0f;
#pragma unroll
        for (int t = 0; t < TS; ++t) {
            w[t] *= scale;
            into[t] *= sigma;
        }
        sigma = kept ? decayed : 1.0f;

        T* o_front = op + t0 * a.out.step;
        const auto o_rows = __builtin_amdgcn_make_buffer_rsrc(o_front, 0, 0x7fffffff, 0x00020000);
        Quad q[TS][NK], p[TS][TS], p_rest[TS][TS];     // [step tile][...]; scores: four y in registers, x in lanes
        if (!LOCAL) {
#pragma unroll
            for (int t = 0; t < TS; ++t)
#pragma unroll
                for (int c = 0; c < NK / 2; ++c) L::row_quads(qs, RK::PITCH, 16 * t + i, c, q[t][2 * c], q[t][2 * c + 1]);
            if constexpr (NK & 1) q[0][NK - 1] = L::row_quad(qs, RK::PITCH, i, NK - 1);
#pragma unroll
            for (int ky = 0; ky < TS; ++ky) {
                __builtin_amdgcn_sched_barrier(0);
                Quad k[NK];
#pragma unroll
                for (int c = 0; c < NK / 2; ++c) L::row_quads(ks, RK::PITCH, 16 * ky + i, c, k[2 * c], k[2 * c + 1]);
                if constexpr (NK & 1) k[NK - 1] = L::row_quad(ks, RK::PITCH, i, NK - 1);
#pragma unroll
                for (int t = 0; t < TS; ++t) {
                    f32x4 z = {0.0f, 0.0f, 0.0f, 0.0f};
                    if (BACK ? t <= ky : t >= ky) {        // (else no pair of these tiles is in order)
#pragma unroll
                        for (int c = 0; c < NK - 1; c += 2) z = L::mma(k[c], k[c + 1], q[t][c], q[t][c + 1], z);
                        if constexpr (NK & 1) z = L::over_steps({k[NK - 1]}, {q[t][NK - 1]}, z);
                        z *= near_of[BACK ? ky - t : t - ky][lane];
                        if (st) {
                            const int g4 = here(4 * g);
                            const uint32_t upto = (2u << here(16 * t + i)) - 1u, cuts = BACK ? st & ~upto : st & upto;
                            const int lo = !BACK && cuts ? 31 - __clz(cuts) : 0, hi = BACK && cuts ? __ffs(cuts) - 1 : CH;
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                const int y = 16 * ky + g4 + r;
                                z[r] = y >= lo && y < hi ? z[r] : 0.0f;
                            }
                        }
                    }
                    p[t][ky] = L::round(z);
                    if (L::SPLIT) p_rest[t][ky] = L::round(z - L::wide(p[t][ky]));
                }
            }
        }

        __builtin_amdgcn_sched_barrier(0);
        uint32_t o_at[TS];                        // a lane's place in the output's rows; behind everything for steps that are not
#pragma unroll
        for (int t = 0; t < TS; ++t) {
            const int step = here(16 * t + i);
            o_at[t] = step < rows ? ((uint32_t)step * (uint32_t)a.out.step + 4 * g) * (uint32_t)sizeof(T) : 0xffffffffu;
        }
        Quad kc[NK][TS];
#pragma unroll
        for (int t = 0; t < TS; ++t)
#pragma unroll
            for (int c = 0; c < NK; ++c) kc[c][t] = L::state_column(ks, RK::PITCH, 16 * t, c);
        __builtin_amdgcn_sched_barrier(0);
        if (x + 1 < chunks) fetch(x + 1);         // (behind the scores: their operands and the rows in flight do not fit together)
#pragma unroll
        for (int m = 0; m < NV; ++m) {
            __builtin_amdgcn_sched_barrier(0);    // (16 columns at a time: their intermediates are a quarter of the registers)
            Quad v[TS];
#pragma unroll
            for (int t = 0; t < TS; ++t) v[t] = L::value_column(vs, RV::PITCH, 16 * t, m);
            if (!LOCAL) {
                f32x4 o[TS];
#pragma unroll
                for (int t = 0; t < TS; ++t) o[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int c = 0; c < NK - 1; c += 2) {
                    const Quad s0 = L::round(S[c][m]), s1 = L::round(S[c + 1][m]);
#pragma unroll
                    for (int t = 0; t < TS; ++t) o[t] = L::mma(s0, s1, q[t][c], q[t][c + 1], o[t]);
                    if (L::SPLIT) {
                        const Quad r0 = L::round(S[c][m] - L::wide(s0)), r1 = L::round(S[c + 1][m] - L::wide(s1));
#pragma unroll
                        for (int t = 0; t < TS; ++t) o[t] = L::mma(r0, r1, q[t][c], q[t][c + 1], o[t]);
                    }
                }
                if constexpr (NK & 1) o[0] = L::over_steps({S[NK - 1][m]}, {q[0][NK - 1]}, o[0]);
#pragma unroll
                for (int t = 0; t < TS; ++t) {
                    o[t] = L::over_steps(v, p[t], o[t] * into[t]);
                    if (L::SPLIT) o[t] = L::over_steps(v, p_rest[t], o[t]);
                    const int step = 16 * t + i, col = m * 16 + 4 * g;
#pragma unroll
                    for (int r = 0; r < 4; ++r) odd += o[t][r] * 0.0f;       // NaN from anything that is not a finite number
                    if constexpr (VEC) {
                        // a buffer store, which drops a lane whose offset is behind the buffer: behind a branch the stores could not be
                        // counted, and the wait for the next chunk's rows would be one for these as well
                        store_quad(o_rows, here(col) < cols ? o_at[t] : 0xffffffffu, m * 16 * (int)sizeof(T), L::round(o[t]));
                    } else if (step < rows) {
                        T* to = o_front + step * a.out.step + col;
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (col + r < cols) to[r] = from_f32<T>(o[t][r]);
                    }
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            if (!kept) {
#pragma unroll
                for (int c = 0; c < NK; ++c) S[c][m] *= decayed;
            }
            f32x4 rest[TS];
            Quad y[TS];
#pragma unroll
            for (int t = 0; t < TS; ++t) {
                rest[t] = L::wide(v[t]) * w[t];
                y[t] = L::round(rest[t]);
            }
#pragma unroll
            for (int c = 0; c < NK; ++c) S[c][m] = L::over_steps(kc[c], y, S[c][m]);
            if (L::SPLIT) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    if (e == 1 && !a.exact_state) break;
#pragma unroll
                    for (int t = 0; t < TS; ++t) {
                        rest[t] -= L::wide(y[t]);
                        y[t] = L::round(rest[t]);
                    }
#pragma unroll
                    for (int c = 0; c < NK; ++c) S[c][m] = L::over_steps(kc[c], y, S[c][m]);
                }
            }
        }
    }

    if (LOCAL) {
        float* to = a.carry + ((pair * col_tiles + col0 / 16) * a.segs + seg) * (NK * 256);
#pragma unroll
        for (int c = 0; c < NK; ++c)
#pragma unroll
            for (int m = 0; m < NV; ++m)
                if (col0 / 16 + m < col_tiles) *(f32x4*)(to + (m * a.segs * NK + c) * 256 + lane * 4) = S[c][m] * sigma;
        if (lane == 0 && slice == 0) a.through[pair * a.segs + seg] = through;
        return;
    }
    if (a.state_out && seg == a.segs - 1) {
        float* s1 = a.state_out + pair * (int64_t)a.dk * a.dv;
#pragma unroll
        for (int c = 0; c < NK; ++c)
#pragma unroll
            for (int m = 0; m < NV; ++m) {
                const int col = m * 16 + i, row = L::state_row(c, g);
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (col < cols && row + r < a.dk) {
                        const float x = S[c][m][r] * sigma;
                        odd += x * 0.0f;
                        if (a.state_t)
                            s1[(int64_t)(col0 + col) * a.dk + row + r] = x;
                        else
                            s1[(int64_t)(row + r) * a.dv + col0 + col] = x;
                    }
            }
    }
    const bool any = __ballot(odd != 0.0f) != 0;       // (NaN is not 0 either)
    if (lane == 0) a.odd[id] = any ? 1u : 0u;
}

// the states behind a pair's segments, chained: carry[s] = through[s] carry[s - 1] + carry[s]
static __global__ void __launch_bounds__(64) chain_kernel(float* carry, const float* through, int32_t segs, int32_t per, int32_t col_tiles) {
    const int64_t group = blockIdx.y;
    f32x4* c = (f32x4*)(carry + group * segs * per) + blockIdx.x * 64 + threadIdx.x;
    per /= 4;
    const float* p = through + group / col_tiles * segs;
    f32x4 s = c[0];
    int x = 1;
    auto batch = [&](auto n) {                  // loads sent together: behind a store to the same array the compiler sends none ahead
        constexpr int U = decltype(n)::value;
        for (; x + U <= segs - 1; x += U) {
            f32x4 next[U];
            float f[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                next[u] = c[(int64_t)(x + u) * per];
                f[u] = p[x + u];
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                s = f[u] == 0.0f ? next[u] : f[u] * s + next[u];
                c[(int64_t)(x + u) * per] = s;
            }
        }
    };
    batch(std::integral_constant<int, 16>{});
    batch(std::integral_constant<int, 4>{});
    batch(std::integral_constant<int, 1>{});
}

// ---- the recurrence itself, one step after the other, for pairs whose results are not all finite numbers: a product's masked terms
// are zeros, and zero times NaN or infinity is NaN, so in such a pair values may have leaked into steps that do not see them.
// Thread (column c, part p of eight) keeps 16 of the state's rows in registers. ----
template <typename T, bool BACK>
__device__ __forceinline__ void recurrent(const ChunkArgs& a, int64_t pair, int col0, float (&row)[2][kMaxHeadDim]) {
    const int64_t n = pair / a.heads;
    const int h = (int)(pair - n * a.heads);
    const int g = threadIdx.x & 7, c = col0 + (threadIdx.x >> 3);
    const float decay = expf(log_decay_of(a.log_decay, h));
    const float* s0 = a.state ? a.state + pair * (int64_t)a.dk * a.dv : nullptr;
    auto at = [&](int i) { return a.state_t ? (int64_t)c * a.dk + i : (int64_t)i * a.dv + c; };
    float s[16];
#pragma unroll
    for (int x = 0; x < 16; ++x) {
        const int i = x * 8 + g;
        s[x] = s0 && i < a.dk && c < a.dv ? s0[at(i)] : 0.0f;
    }
    auto cut = [&](int64_t t) { return a.starts && a.starts[n * a.starts_batch + t * a.starts_step]; };
    for (int64_t u = 0; u < a.steps; ++u) {
        const int64_t t = BACK ? a.steps - 1 - u : u;
        const T* qp = (const T*)a.q.p + n * a.q.batch + t * a.q.step + h * a.q.head;
        const T* kp = (const T*)a.k.p + n * a.k.batch + t * a.k.step + h * a.k.head;
        const T* vp = (const T*)a.v.p + n * a.v.batch + t * a.v.step + h * a.v.head;
        __syncthreads();
        for (int i = threadIdx.x; i < a.dk; i += 256) {
            row[0][i] = to_f32(qp[i]) * a.read_scale;
            row[1][i] = to_f32(kp[i]) * a.write_scale;
        }
        __syncthreads();
        float keep = decay;
        if (BACK)
            keep = u == 0 ? 1.0f : cut(t + 1) ? 0.0f : decay;
        else if (cut(t))
            keep = 0.0f;
        const float vc = c < a.dv ? to_f32(vp[c]) : 0.0f;
        float o = 0.0f;
#pragma unroll
        for (int x = 0; x < 16; ++x) {
            const int i = x * 8 + g;
            if (i < a.dk) {
                s[x] = (keep == 0.0f ? 0.0f : keep * s[x]) + row[1][i] * vc;
                o += row[0][i] * s[x];
            }
        }
        o += __shfl_xor(o, 1);
        o += __shfl_xor(o, 2);
        o += __shfl_xor(o, 4);
        if (g == 0 && c < a.dv) ((T*)a.out.p)[n * a.out.batch + t * a.out.step + h * a.out.head + c] = from_f32<T>(o);
    }
    if (a.state_out && c < a.dv) {
        float* s1 = a.state_out + pair * (int64_t)a.dk * a.dv;
        const float last = BACK && a.steps > 0 ? (cut(0) ? 0.0f : decay) : 1.0f;
#pragma unroll
        for (int x = 0; x < 16; ++x) {
            const int i = x * 8 + g;
            if (i < a.dk) s1[at(i)] = last == 0.0f ? 0.0f : last * s[x];
        }
    }
}

constexpr int kOddGroup = 64;

template <typename T, bool BACK>
__global__ void __launch_bounds__(256) odd_kernel(ChunkArgs a, int64_t pairs) {
    __shared__ float row[2][kMaxHeadDim];
    __shared__ uint32_t odd[kOddGroup];
    const int per = a.slices * a.segs;
    for (int64_t p0 = (int64_t)blockIdx.x * kOddGroup; p0 < pairs; p0 += (int64_t)gridDim.x * kOddGroup) {
        const int here = pairs - p0 < kOddGroup ? (int)(pairs - p0) : kOddGroup;
        if (threadIdx.x < kOddGroup) odd[threadIdx.x] = 0;
        __syncthreads();
        bool any = false;
        for (int x = threadIdx.x; x < here * per; x += 256)
            if (a.odd[p0 * per + x]) {
                odd[x / per] = 1;
                any = true;
            }
        if (!__syncthreads_or(any)) continue;
        for (int x = 0; x < here; ++x) {
            if (!odd[x]) continue;
            for (int col = 0; col < a.dv; col += 32) recurrent<T, BACK>(a, p0 + x, col, row);
        }
        __syncthreads();
    }
}

// The recurrence for every pair, 32 columns of its state a workgroup, where there are few steps and no more workgroups than the chip
// holds at once: a chunk would be nearly empty.  16 pairs of 32 x 32: 5 us a step, 7 four, chunks 10; 16384 pairs, four steps: 61 us,
// chunks 32; 512 pairs of 128 x 128, the most that take this way: four steps as long as chunks, eight 10 us longer
constexpr int64_t kFewSteps = 8, kFewGroups = 2048;

template <typename T, bool BACK>
__global__ void __launch_bounds__(256) few_steps_kernel(ChunkArgs a) {
    __shared__ float row[2][kMaxHeadDim];
    recurrent<T, BACK>(a, blockIdx.x, blockIdx.y * 32, row);
}

// How a walk over (batch, heads) pairs is cut: column slices of the state, and, where there are few waves and many steps, segments of
// the steps, whose states are computed first (from k and v alone) and chained.
struct WalkPlan {
    int nk, nv, slices, segs;                // tiles of 16 rows and of 16 columns a wave
    int64_t seg_steps;
};

static WalkPlan walk_plan(int32_t dtype, int64_t pairs, int64_t steps, int dk, int dv, bool wide) {
    WalkPlan p;
    p.nk = (int)ceil_div(dk, 16);
    p.nk = p.nk < 2 ? 2 : p.nk == 7 ? 8 : p.nk;
    if (dtype == FISHING_DTYPE_BF16) p.nk += p.nk & 1;
    // columns a wave: as many tiles as multiply the least (each slice computes the scores anew; a tile behind dv is work for nothing);
    // rows that are not whole 16-byte accesses: one width is enough
    p.nv = 2;
    auto cost = [&](int nv) { return ceil_div(dv, 16 * nv) * (p.nk + nv * (2 * p.nk + 1)); };
    for (int nv = 3; nv <= 4 && wide; ++nv)
        if (cost(nv) <= cost(p.nv)) p.nv = nv;
    p.slices = (int)ceil_div(dv, p.nv * 16);
    // Segments: as many waves as 1024 SIMDs hold (three each of the small states), of at least 8 chunks each, for a segment costs a
    // state written, read, chained and read.  (97 x 1009 steps, 3 heads of 48 x 80, f32, with gradients: at least 16 chunks and two
    // waves 666 us, 8 and three 527, 6 and four 565.)
    const bool f32 = dtype == FISHING_DTYPE_F32;
    const int64_t waves = pairs * p.slices, each = p.nk * p.nv <= (f32 ? 9 : 6) ? 3 : waves_a_simd(p.nk, p.nv, wide, false);
    const int64_t want = waves > 0 ? 1024 * each / waves : 1, most = steps / (f32 ? 128 : 256);
    int64_t segs = want < most ? want : most;
    if (segs < 2) segs = 1;
    p.seg_steps = segs > 1 ? round_up(ceil_div(steps, segs), 32) : (steps > 0 ? steps : 1);
    p.segs = steps > 0 ? (int)ceil_div(steps, p.seg_steps) : 1;
    return p;
}

template <int N>
using Count = std::integral_constant<int, N>;

struct WalkWork {
    float *carry, *through;
    uint32_t* odd;
    int64_t bytes;
};

static WalkWork walk_work(const WalkPlan& p, int64_t pairs, int dv, float* carry, void* at) {
    Carve c(at);
    WalkWork w{};
    w.odd = c.take<uint32_t>(pairs * p.slices * p.segs);
    w.carry = carry;
    if (p.segs > 1 && !carry) {
        w.through = c.take<float>(pairs * p.segs);
        w.carry = c.take<float>(pairs * ceil_div(dv, 16) * p.segs * p.nk * 256);
    }
    w.bytes = round_up(c.used, 256);
    return w;
}

// What a walk in segments leaves to one whose state is its own transposed, from the same terms: the states it starts its segments from
struct Shared {
    bool exact = false;        // the other's state is an answer
    int nk = 0, segs = 1;
    int64_t seg_steps = 0;
    float* carry = nullptr;
    int64_t bytes = 0;         // of the workspace, not to be written
};

template <typename T, bool BACK>
int walk(const FishingDecayAttention* f, Strided q, Strided k, Strided v, const float* state, float* state_out, Strided out, int dk, int dv, bool state_t, bool exact_state,
                double read_scale, double write_scale, Shared* shared, void* workspace, hipStream_t stream) {
    if (f->steps <= 1) q.step = k.step = v.step = out.step = kMaxHeadDim;         // (a single step has no next one: any stride will do)
    constexpr int V = vec_of<T>();
    auto wide = [&](const Strided& s, int d) {
        return d % V == 0 && aligned16(s.p) && s.batch % V == 0 && s.step % V == 0 && s.head % V == 0 && s.step >= d && s.step < (int64_t)1 << 24;
    };
    const bool vec = wide(q, dk) && wide(k, dk) && wide(v, dv) && wide(out, dv) && f->starts_stride[1] >= 0 && f->starts_stride[1] < (int64_t)1 << 24;
    const int64_t block = batch_block(f->batch, f->heads);
    WalkPlan p = walk_plan(f->dtype, block * f->heads, f->steps, dk, dv, vec);
    const bool given = shared && shared->nk;
    if (given) {
        p.segs = shared->segs;
        p.seg_steps = shared->seg_steps;
    } else if (shared) {                        // (of the two plans the one of fewer segments)
        const WalkPlan other = walk_plan(f->dtype, block * f->heads, f->steps, dv, dk, vec);
        if (other.segs > 1 && other.segs < p.segs) {
            p.segs = other.segs;
            p.seg_steps = other.seg_steps;
        }
    }
    const WalkWork w = walk_work(p, block * f->heads, dv, given ? shared->carry : nullptr, (char*)workspace + (given ? shared->bytes : 0));
    if (shared && !given && p.segs > 1) *shared = Shared{shared->exact, p.nk, p.segs, p.seg_steps, w.carry, w.bytes};
    ChunkArgs a{q, k, v, out, f->log_decay, f->starts, f->starts_stride[0], f->starts_stride[1], state, state_out, f->steps, f->heads, dk, dv, state_t, exact_state,
                      (float)read_scale, (float)write_scale, p.slices, p.segs, p.seg_steps, w.carry, w.through, w.odd, given ? shared->nk : 0};
    int64_t pairs = 0;
    auto run = [&](auto tk, auto tv, auto rows) {
        const dim3 grid((unsigned)(pairs * p.slices * p.segs));
        constexpr int NK = decltype(tk)::value, NV = decltype(tv)::value;
        constexpr bool VEC = decltype(rows)::value;
        int rc = 0;
        if (p.segs > 1 && !given) {
            // without outputs narrow slices fit two waves on a SIMD (16381 steps, 8 heads of 128 x 128: 26 us, with 4 tiles 44)
            constexpr int LV = NK >= 5 ? 2 : NV;
            const int per = NK * 256, col_tiles = (int)ceil_div(dv, 16);
            ChunkArgs local = a;
            local.slices = (int)ceil_div(dv, LV * 16);
            local.exact_state = exact_state || (shared && shared->exact);
            rc = launch(chunk_kernel<T, NK, LV, BACK, VEC, true>, dim3((unsigned)(pairs * local.slices * p.segs)), dim3(64), stream, local);
            if (!rc) rc = launch(chain_kernel, dim3((unsigned)(per / 256), (unsigned)(pairs * col_tiles)), dim3(64), stream, w.carry, w.through, p.segs, per, col_tiles);
        }
        return rc ? rc : launch(chunk_kernel<T, NK, NV, BACK, VEC, false>, grid, dim3(64), stream, a);
    };
    auto tiles = [&](auto tv, auto rows) {
        if constexpr (sizeof(T) == 4) {
            if (p.nk == 3) return run(Count<3>{}, tv, rows);
            if (p.nk == 5) return run(Count<5>{}, tv, rows);
        }
        return p.nk == 2 ? run(Count<2>{}, tv, rows) : p.nk == 4 ? run(Count<4>{}, tv, rows) : p.nk == 6 ? run(Count<6>{}, tv, rows) : run(Count<8>{}, tv, rows);
    };
    int rc = 0;
    for (int64_t n = 0; n < f->batch && !rc; n += block) {
        pairs = (f->batch - n < block ? f->batch - n : block) * f->heads;
        if (f->steps <= kFewSteps && pairs * ceil_div(dv, 32) <= kFewGroups) {
            rc = launch(few_steps_kernel<T, BACK>, dim3((unsigned)pairs, (unsigned)ceil_div(dv, 32)), dim3(256), stream, a);
        } else {
            rc = !vec ? tiles(Count<2>{}, std::false_type{}) : p.nv == 2 ? tiles(Count<2>{}, std::true_type{}) : p.nv == 3 ? tiles(Count<3>{}, std::true_type{}) : tiles(Count<4>{}, std::true_type{});
            const int64_t groups = ceil_div(pairs, kOddGroup);
            if (!rc) rc = launch(odd_kernel<T, BACK>, dim3((unsigned)(groups < 1024 ? groups : 1024)), dim3(256), stream, a, pairs);
        }
        if (rc) break;
        // the next block's corners
        for (Strided* s : {&a.q, &a.k, &a.v, &a.out}) s->p = (const T*)s->p + block * s->batch;
        if (a.starts) a.starts += block * a.starts_batch;
        if (a.state) a.state += block * f->heads * dk * dv;
        if (a.state_out) a.state_out += block * f->heads * dk * dv;
    }
    return rc;
}

}  // namespace seq
}  // namespace fishing
