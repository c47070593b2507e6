// sequence_embedding.hip -- rows of a table for tokens, and the table's gradient by sorted tokens.
#include "sequence_common.h"

namespace fishing {
namespace seq {

// out[i] = scale * table[token[i]]; a token outside [0, vocab) is padding: a row of zeros.
// A block owns 256 / vecs rows at a time (vecs accesses a row), four times over, so that four rows' loads are in flight; bound by the
// rows written: 1034240 x 256 f32 220 us, 4.8 TB/s; 413696 x 128 bf16 23 us, 4.6 TB/s; 4096 x 64 bf16 4 us, the launch's own.
template <typename T, typename I, int V, bool PAST>
__global__ void __launch_bounds__(256) embedding_kernel(const T* table, int64_t table_stride, const I* token, int64_t n, int64_t vocab,
                                                        int32_t vecs, float scale, T* out) {
    const int per = vecs < 256 ? 256 / vecs : 1;
    const int r = threadIdx.x / vecs < per ? threadIdx.x / vecs : -1;
    const int c0 = vecs < 256 ? threadIdx.x % vecs : threadIdx.x;
    if (vecs < 256 && r < 0) return;
    const int64_t dim = (int64_t)vecs * V;
#pragma unroll 4
    for (int j = 0; j < 4; ++j) {
        const int64_t i = ((int64_t)blockIdx.x * 4 + j) * per + (vecs < 256 ? r : 0);
        if (i >= n) return;
        const int64_t t = (int64_t)token[i];
        const bool there = t >= 0 && t < vocab;
        for (int c = c0; c < vecs; c += 256) {
            Pack<T, V> x;
            if (there) {
                x = *(const Pack<T, V>*)(table + t * table_stride + (int64_t)c * V);
#pragma unroll
                for (int e = 0; e < V; ++e) x.e[e] = from_f32<T>(to_f32(x.e[e]) * scale);
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e) x.e[e] = from_f32<T>(0.0f);
            }
            typedef typename std::conditional<(V > 1), u32x4, T>::type Access;
            Access* to = (Access*)(out + i * dim + (int64_t)c * V);
            if constexpr (PAST)
                __builtin_nontemporal_store(*(Access*)&x, to);
            else
                *to = *(Access*)&x;
        }
    }
}

// ---- the gradient: dtable[v] = scale * sum of dout[i] over the i with token[i] == v, in ascending i ----
// A stable radix sort of (token, i) by up to 8 bits a pass puts a token's rows side by side; then chunks of the sorted order
// are summed in float32 registers, and runs that cross a chunk's border leave a partial row that the last kernel adds in
// chunk order.  No atomics on sums: the same bits every time.  Bound by the rows read once, in the tokens' order: 1034240 x 256 f32,
// 100 tokens: sorting 23 us, sums 206 (5.1 TB/s), join 10; 413696 x 128 bf16, 10001 tokens, two passes: sorting 29, sums 38
// (2.8 TB/s: runs are 40 rows long), join 10.  (A table of partial sums in LDS, for few tokens, took 452 us where this takes 240; its
// float atomics 1354.)
constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / 64, kMaxDigits = 256;

__device__ __forceinline__ uint32_t key_of(int64_t t, int64_t vocab) { return t >= 0 && t < vocab ? (uint32_t)t : (uint32_t)vocab; }

template <typename I, bool FIRST>
__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(const I* token, const uint32_t* key, int64_t n, int64_t vocab, int64_t tile, int shift,
                                                                  int digits, uint32_t* count) {
    __shared__ uint32_t bin[kMaxDigits];
    for (int d = threadIdx.x; d < digits; d += kSortThreads) bin[d] = 0;
    __syncthreads();
    const int64_t lo = (int64_t)blockIdx.x * tile, hi = lo + tile < n ? lo + tile : n;
    for (int64_t i = lo + threadIdx.x; i < hi; i += kSortThreads) {
        const uint32_t k = FIRST ? key_of((int64_t)token[i], vocab) : key[i];
        atomicAdd(&bin[(k >> shift) & (digits - 1)], 1u);   // whole numbers: the order does not matter
    }
    __syncthreads();
    for (int d = threadIdx.x; d < digits; d += kSortThreads) count[(int64_t)d * gridDim.x + blockIdx.x] = bin[d];
}

constexpr int kMaxBlocks = 512;

// a workgroup per digit: its blocks' counts become exclusive sums, count[digits * blocks + digit] their total
__global__ void __launch_bounds__(kMaxBlocks) sort_scan_kernel(uint32_t* count, int32_t blocks, int32_t digits) {
    __shared__ uint32_t sum[kMaxBlocks / 64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    uint32_t* c = count + (int64_t)blockIdx.x * blocks;
    const uint32_t mine = threadIdx.x < (uint32_t)blocks ? c[threadIdx.x] : 0;
    uint32_t s = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t x = __shfl_up(s, d);
        if (lane >= d) s += x;
    }
    if (lane == 63) sum[wave] = s;
    __syncthreads();
    for (int w = 0; w < wave; ++w) s += sum[w];
    if (threadIdx.x < (uint32_t)blocks) c[threadIdx.x] = s - mine;
    if (threadIdx.x == kMaxBlocks - 1) count[(int64_t)digits * blocks + blockIdx.x] = s;
}

template <typename I, bool FIRST>
__global__ void __launch_bounds__(kSortThreads) sort_place_kernel(const I* token, const uint32_t* key, const uint32_t* row, int64_t n, int64_t vocab,
                                                                  int64_t tile, int shift, int bits, const uint32_t* count, uint32_t* key_out, uint32_t* row_out) {
    __shared__ uint32_t base[kMaxDigits];
    __shared__ uint32_t in_wave[kSortWaves][kMaxDigits];
    const int digits = 1 << bits, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    // where this block's share of each digit begins: the digits before it, and the blocks before this one
    if (threadIdx.x < kMaxDigits) {
        const uint32_t total = threadIdx.x < (uint32_t)digits ? count[(int64_t)digits * gridDim.x + threadIdx.x] : 0;
        uint32_t s = total;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t x = __shfl_up(s, d);
            if (lane >= d) s += x;
        }
        if (lane == 63) in_wave[0][wave] = s;
        base[threadIdx.x] = s - total;
    }
    __syncthreads();
    if (threadIdx.x < (uint32_t)digits) {
        uint32_t s = base[threadIdx.x] + count[(int64_t)threadIdx.x * gridDim.x + blockIdx.x];
        for (int w = 0; w < wave; ++w) s += in_wave[0][w];
        base[threadIdx.x] = s;
    }
    __syncthreads();
    const int64_t lo = (int64_t)blockIdx.x * tile, hi = lo + tile < n ? lo + tile : n;
    for (int64_t i0 = lo; i0 < hi; i0 += kSortThreads) {
        for (int d = threadIdx.x; d < kSortWaves * digits; d += kSortThreads) in_wave[d >> bits][d & (digits - 1)] = 0;
        __syncthreads();
        const int64_t i = i0 + threadIdx.x;
        const bool there = i < hi;
        uint32_t k = 0, from = 0;
        if (there) {
            k = FIRST ? key_of((int64_t)token[i], vocab) : key[i];
            from = FIRST ? (uint32_t)i : row[i];
        }
        const uint32_t d = (k >> shift) & (digits - 1);
        uint64_t same = __ballot(there);
        for (int b = 0; b < bits; ++b) {
            const uint64_t set = __ballot((d >> b) & 1);
            same &= (d >> b) & 1 ? set : ~set;
        }
        const uint32_t rank = __popcll(same & ((1ull << lane) - 1));
        if (there && rank == 0) in_wave[wave][d] = __popcll(same);
        __syncthreads();
        for (int x = threadIdx.x; x < digits; x += kSortThreads) {
            uint32_t run = base[x];
            for (int w = 0; w < kSortWaves; ++w) {
                const uint32_t c = in_wave[w][x];
                in_wave[w][x] = run;
                run += c;
            }
            base[x] = run;
        }
        __syncthreads();
        if (there) {
            const uint32_t at = in_wave[wave][d] + rank;
            key_out[at] = k;
            row_out[at] = from;
        }
        __syncthreads();
    }
}

// start[v] = first sorted position with a key >= v, v = 0 .. vocab; written where the key changes, by the lanes of a group
template <int G>
__device__ __forceinline__ void mark_starts(uint32_t* start, int64_t from, int64_t to, uint32_t at, int lane) {
    for (int64_t v = from + lane; v <= to; v += G) start[v] = at;
}

// A group of G lanes sums one chunk of the sorted order, V columns a lane; blockIdx.y walks the columns beyond G * V.
template <typename T, int V, int G>
__global__ void __launch_bounds__(256) embedding_sum_kernel(const T* dout, int64_t dout_stride, const uint32_t* key, const uint32_t* row, int64_t n, int64_t vocab,
                                                            int32_t dim, int32_t chunk, float scale, T* dtable, float* partial, uint32_t* start) {
    constexpr int U = 16;
    const int lane = threadIdx.x % G;
    const int64_t c = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
    const int64_t p0 = c * chunk, p1 = p0 + chunk < n ? p0 + chunk : n;
    if (p0 >= n) return;
    const int col = (blockIdx.y * G + lane) * V;
    const bool mine = col < dim, marks = blockIdx.y == 0;
    const int64_t before = p0 > 0 ? (int64_t)key[p0 - 1] : -1, after = p1 < n ? (int64_t)key[p1] : -1;
    float acc[V];
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] = 0.0f;
    int64_t cur = key[p0];
    bool first = true;
    if (marks && cur != before) mark_starts<G>(start, before + 1, cur, (uint32_t)p0, lane);
    auto flush = [&](bool last) {
        if (cur < vocab && mine) {
            const bool crosses = (first && cur == before) || (last && cur == after);
            if (crosses) {
                float* to = partial + (2 * c + (first ? 0 : 1)) * dim + col;
#pragma unroll
                for (int e = 0; e < V; ++e) to[e] = acc[e];
            } else {
                Pack<T, V> x;
#pragma unroll
                for (int e = 0; e < V; ++e) x.e[e] = from_f32<T>(acc[e] * scale);
                *(Pack<T, V>*)(dtable + cur * dim + col) = x;
            }
        }
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] = 0.0f;
        first = false;
    };
    uint32_t k[U], from[U];
    auto index = [&](int64_t p) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t at = p + u < p1 ? p + u : p1 - 1;
            k[u] = key[at];
            from[u] = row[at];
        }
    };
    index(p0);
    for (int64_t p = p0; p < p1; p += U) {
        uint32_t now[U];
        Pack<T, V> x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            now[u] = k[u];
            if (mine && now[u] < vocab) x[u] = *(const Pack<T, V>*)(dout + (int64_t)from[u] * dout_stride + col);
        }
        if (p + U < p1) index(p + U);              // (the next rows' places arrive with this batch's rows)
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (p + u < p1) {
                if ((int64_t)now[u] != cur) {
                    flush(false);
                    if (marks) mark_starts<G>(start, cur + 1, now[u], (uint32_t)(p + u), lane);
                    cur = now[u];
                }
                if (mine && now[u] < vocab) {
#pragma unroll
                    for (int e = 0; e < V; ++e) acc[e] += to_f32(x[u].e[e]);
                }
            }
        }
    }
    flush(true);
    if (marks && p1 == n) mark_starts<G>(start, cur + 1, vocab, (uint32_t)n, lane);
}

// the rows the chunks did not finish: tokens that were never met (zeros) and runs over several chunks (their partials' sum)
// A run's partials are one chain of additions, 8 loads ahead: 10 us where a token has a hundred of them, and nearly all of the gradient's
// 613 us where 2^20 rows of 8 bf16 are two tokens' (16384 partials each), or of 781 where they are one's and 128 wide.
template <typename T>
__global__ void __launch_bounds__(256) embedding_join_kernel(const uint32_t* start, const float* partial, int64_t n, int64_t vocab, int32_t dim, int32_t chunk,
                                                             float scale, T* dtable) {
    for (int64_t v = blockIdx.x; v < vocab; v += gridDim.x) {
        const int64_t s = n ? start[v] : 0, e = n ? start[v + 1] : 0;
        const int64_t a = s / chunk, b = e > s ? (e - 1) / chunk : a;
        if (e > s && a == b) continue;
        for (int col = threadIdx.x; col < dim; col += 256) {
            float acc = 0.0f;
            if (e > s) {
                acc = partial[(2 * a + (s == a * chunk ? 0 : 1)) * dim + col];
#pragma unroll 8
                for (int64_t c = a + 1; c <= b; ++c) acc += partial[2 * c * dim + col];
            }
            dtable[v * dim + col] = from_f32<T>(acc * scale);
        }
    }
}

// ---- the same for few tokens, in one launch: a workgroup per `rows` of the table and 32 lanes of columns lists the tokens that are a row's,
// in their order; groups of lanes sum shares of the list, which are added in order.  Bound by a few trips to memory after each other, and
// by every workgroup's look at every token: 2048 tokens, 101 x 64 f32: 8 us, sorted 19; 10001 x 128: 22, 36; 16 x 512: 11, 19; 131072 x 64:
// 30, 136; 2^20 x 64: 122, 576; 2^24 x 8 bf16: 1390, 7850 (a look at every row of the table either way).  4096: 101 x 64 13, 20;
// 10001 x 128 40, 36; so up to 4096 tokens where a workgroup has one row, else 2048
constexpr int kDirectTokens = 4096, kDirectVocab = 2048, kDirectRows = 16, kDirectLanes = 32;

template <typename T, typename I, int V>
__global__ void __launch_bounds__(256) embedding_direct_kernel(const T* dout, int64_t dout_stride, const I* token, int32_t n, int64_t vocab, int32_t dim, int32_t rows,
                                                               float scale, T* dtable) {
    __shared__ uint32_t met;
    __shared__ int in_wave[4];
    __shared__ uint16_t list[kDirectTokens];
    __shared__ float part[256][V + 1];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t v0 = (int64_t)blockIdx.x * rows;
    const int rows_here = vocab - v0 < rows ? (int)(vocab - v0) : rows;
    const int lanes_left = dim / V - (int)blockIdx.y * kDirectLanes, lanes = lanes_left < kDirectLanes ? lanes_left : kDirectLanes, groups = 256 / lanes;
    const int g = threadIdx.x / lanes, c = threadIdx.x % lanes;
    T* to = dtable + v0 * dim + ((int)blockIdx.y * kDirectLanes + c) * V;
    if (threadIdx.x == 0) met = 0;
    __syncthreads();
    uint32_t mine = 0;
    for (int i = threadIdx.x; i < n; i += 256) {
        const int64_t r = (int64_t)token[i] - v0;
        if (r >= 0 && r < rows_here) mine |= 1u << r;
    }
    if (mine) atomicOr(&met, mine);
    __syncthreads();
    const uint32_t has = met;
    Pack<T, V> zero;
#pragma unroll
    for (int e = 0; e < V; ++e) zero.e[e] = from_f32<T>(0.0f);
    for (int r = g; r < rows_here; r += groups)
        if (g < groups && !(has >> r & 1)) *(Pack<T, V>*)(to + (int64_t)r * dim) = zero;
    for (int r = 0; r < rows_here; ++r) {
        if (!(has >> r & 1)) continue;
        int total = 0;
        for (int i0 = 0; i0 < n; i0 += 256) {
            const int i = i0 + threadIdx.x;
            const bool hit = i < n && (int64_t)token[i] == v0 + r;
            const uint64_t all = __ballot(hit);
            if (lane == 0) in_wave[wave] = __popcll(all);
            __syncthreads();
            int at = total;
            for (int w = 0; w < wave; ++w) at += in_wave[w];
            if (hit) list[at + __popcll(all & ((1ull << lane) - 1))] = (uint16_t)i;
            total += in_wave[0] + in_wave[1] + in_wave[2] + in_wave[3];
            __syncthreads();
        }
        const int share = (total + groups - 1) / groups, lo = g * share, hi = lo + share < total ? lo + share : total;
        float acc[V];
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] = 0.0f;
        if (g < groups) {
#pragma unroll 8
            for (int x = lo; x < hi; ++x) {
                const Pack<T, V> y = *(const Pack<T, V>*)(dout + (int64_t)list[x] * dout_stride + ((int)blockIdx.y * kDirectLanes + c) * V);
#pragma unroll
                for (int e = 0; e < V; ++e) acc[e] += to_f32(y.e[e]);
            }
        }
#pragma unroll
        for (int e = 0; e < V; ++e) part[threadIdx.x][e] = acc[e];
        __syncthreads();
        if (g == 0) {
            const int with = (total + share - 1) / share;              // groups that had a share
            for (int x = 1; x < with; ++x) {
#pragma unroll
                for (int e = 0; e < V; ++e) acc[e] += part[x * lanes + c][e];
            }
            Pack<T, V> y;
#pragma unroll
            for (int e = 0; e < V; ++e) y.e[e] = from_f32<T>(acc[e] * scale);
            *(Pack<T, V>*)(to + (int64_t)r * dim) = y;
        }
        __syncthreads();
    }
}

struct SortPlan {
    int bits, passes, digit_bits;
    int64_t tile;
    int blocks;
    int32_t chunk;
    int64_t chunks;
};

static SortPlan sort_plan(int64_t n, int64_t vocab, int64_t lanes) {
    SortPlan s;
    s.bits = 1;
    while (((int64_t)1 << s.bits) <= vocab) ++s.bits;         // keys 0 .. vocab
    s.passes = (s.bits + 7) / 8;
    s.digit_bits = (s.bits + s.passes - 1) / s.passes;
    s.tile = round_up(ceil_div(n > 0 ? n : 1, kMaxBlocks), 2 * kSortThreads);
    s.blocks = (int)ceil_div(n > 0 ? n : 1, s.tile);
    // A chunk is a group's: so long that about 4096 waves of groups share the rows (64 waves' worth of rows in flight on every CU; 1034240
    // rows of 256 f32: 256 rows a chunk 257 us with the join, 64 292; 413696 rows of 128 bf16: 64 49 us, 256 157), within 16 .. 256
    const int64_t group = lanes <= 8 ? 8 : lanes <= 16 ? 16 : lanes <= 32 ? 32 : 64;
    s.chunk = 16;
    while (s.chunk < 256 && s.chunk * 4096 * (64 / group) < n * ceil_div(lanes, 64)) s.chunk *= 2;
    s.chunks = ceil_div(n, s.chunk);
    return s;
}

struct EmbeddingWork {
    uint32_t *key[2], *row[2], *count, *start;
    float* partial;
    int64_t bytes;
};

static EmbeddingWork embedding_work(const SortPlan& s, int64_t n, int64_t vocab, int64_t dim, void* at) {
    Carve c(at);
    EmbeddingWork w;
    for (int k = 0; k < 2; ++k) {
        w.key[k] = c.take<uint32_t>(n);
        w.row[k] = c.take<uint32_t>(n);
    }
    w.count = c.take<uint32_t>((int64_t)(s.blocks + 1) << s.digit_bits);
    w.start = c.take<uint32_t>(vocab + 1);
    w.partial = c.take<float>(2 * s.chunks * dim);
    w.bytes = c.used;
    return w;
}

// lanes that a row takes in 16-byte accesses
static int64_t row_lanes(int32_t dtype, int64_t dim) { return ceil_div(dim, dtype == FISHING_DTYPE_F32 ? 4 : 8); }

static int embedding_check(int32_t dtype, int32_t index_bytes, int64_t n, int64_t vocab, int64_t dim) {
    if (dtype != FISHING_DTYPE_F32 && dtype != FISHING_DTYPE_BF16) return FISHING_ERR_UNSUPPORTED;
    if (index_bytes != 4 && index_bytes != 8) return FISHING_ERR_UNSUPPORTED;
    if (n < 0 || n > 0x7fffffff || vocab < 1 || vocab > 0x7ffffffe || dim < 1 || dim > 65536) return FISHING_ERR_SIZE;
    return FISHING_OK;
}

// Rows that the 256 MiB of cache in front of HBM cannot hold for their reader are written past it, and what it holds stays: 1034240 rows
// of 256 f32, forward and backward: 435 us, 500 through it.  Rows that fit are left there
constexpr int64_t kPastCaches = (int64_t)256 << 20;
constexpr int64_t kMaxGrid = (int64_t)1 << 22;      // workgroups of 256, whose threads count in 32 bits

template <typename T, typename I>
static int embedding_forward(int64_t n, int64_t vocab, int64_t dim, const T* table, int64_t table_stride, const I* token, float scale, T* out, hipStream_t stream) {
    constexpr int V = vec_of<T>();
    auto go = [&](auto kernel, int vecs) {
        const int64_t block = (vecs < 256 ? 256 / vecs : 1) * 4 * kMaxGrid;       // rows of a launch
        int rc = 0;
        for (int64_t i = 0; i < n && !rc; i += block) {
            const int64_t here = n - i < block ? n - i : block;
            rc = launch(kernel, dim3((unsigned)ceil_div(here, block / kMaxGrid)), dim3(256), stream, table, table_stride, token + i, here, vocab, vecs, scale, out + i * dim);
        }
        return rc;
    };
    const bool past = n * dim * (int64_t)sizeof(T) >= kPastCaches;
    if (dim % V == 0 && table_stride % V == 0 && aligned16(table) && aligned16(out))
        return past ? go(embedding_kernel<T, I, V, true>, (int)(dim / V)) : go(embedding_kernel<T, I, V, false>, (int)(dim / V));
    return go(embedding_kernel<T, I, 1, false>, (int)dim);
}

template <typename T, typename I>
static int embedding_backward(int64_t n, int64_t vocab, int64_t dim, const T* dout, int64_t dout_stride, const I* token, float scale, T* dtable, void* workspace,
                              hipStream_t stream) {
    if (n <= (vocab <= kDirectVocab ? kDirectTokens : kDirectTokens / 2) && ceil_div(vocab, kDirectRows) <= kMaxGrid) {
        const int64_t few = ceil_div(vocab, kDirectVocab), rows = few < kDirectRows ? few : kDirectRows;
        auto direct = [&](auto kernel, int v) {
            const int64_t across = ceil_div(dim / v, kDirectLanes), blocks = ceil_div(vocab, rows);
            return launch(kernel, dim3((unsigned)blocks, (unsigned)across), dim3(256), stream, dout, dout_stride, token, (int32_t)n, vocab, (int32_t)dim, (int32_t)rows, scale, dtable);
        };
        constexpr int V = vec_of<T>();
        return dim % V == 0 && dout_stride % V == 0 && aligned16(dout) && aligned16(dtable) ? direct(embedding_direct_kernel<T, I, V>, V) : direct(embedding_direct_kernel<T, I, 1>, 1);
    }
    int rc = 0;
    const SortPlan s = sort_plan(n, vocab, row_lanes(sizeof(T) == 4 ? FISHING_DTYPE_F32 : FISHING_DTYPE_BF16, dim));
    const EmbeddingWork w = embedding_work(s, n, vocab, dim, workspace);
    if (n > 0) {
        for (int p = 0; p < s.passes && !rc; ++p) {
            const int shift = p * s.digit_bits, digits = 1 << s.digit_bits;
            const uint32_t *key = w.key[(p + 1) & 1], *row = w.row[(p + 1) & 1];
            const dim3 grid(s.blocks), block(kSortThreads);
            rc = p == 0 ? launch(sort_count_kernel<I, true>, grid, block, stream, token, key, n, vocab, s.tile, shift, digits, w.count)
                        : launch(sort_count_kernel<I, false>, grid, block, stream, token, key, n, vocab, s.tile, shift, digits, w.count);
            if (!rc) rc = launch(sort_scan_kernel, dim3(digits), dim3(kMaxBlocks), stream, w.count, s.blocks, digits);
            if (!rc)
                rc = p == 0 ? launch(sort_place_kernel<I, true>, grid, block, stream, token, key, row, n, vocab, s.tile, shift, s.digit_bits, w.count, w.key[0], w.row[0])
                            : launch(sort_place_kernel<I, false>, grid, block, stream, token, key, row, n, vocab, s.tile, shift, s.digit_bits, w.count, w.key[p & 1], w.row[p & 1]);
        }
        if (rc) return rc;
        const uint32_t *key = w.key[(s.passes - 1) & 1], *row = w.row[(s.passes - 1) & 1];
        auto sum = [&](auto kernel, int V, int G) {
            return launch(kernel, dim3((unsigned)ceil_div(s.chunks, 256 / G), (unsigned)ceil_div(dim, G * V)), dim3(256), stream, dout, dout_stride, key, row, n, vocab,
                          (int32_t)dim, s.chunk, scale, dtable, w.partial, w.start);
        };
        constexpr int V = vec_of<T>();
        if (dim % V == 0 && dout_stride % V == 0 && aligned16(dout) && aligned16(dtable)) {
            const int64_t lanes = dim / V;
            rc = lanes <= 8 ? sum(embedding_sum_kernel<T, V, 8>, V, 8) : lanes <= 16 ? sum(embedding_sum_kernel<T, V, 16>, V, 16)
               : lanes <= 32 ? sum(embedding_sum_kernel<T, V, 32>, V, 32) : sum(embedding_sum_kernel<T, V, 64>, V, 64);
        } else {
            rc = sum(embedding_sum_kernel<T, 1, 64>, 1, 64);
        }
        if (rc) return rc;
    }
    return launch(embedding_join_kernel<T>, dim3((unsigned)(vocab < kMaxGrid ? vocab : kMaxGrid)), dim3(256), stream, w.start, w.partial, n, vocab, (int32_t)dim, s.chunk, scale, dtable);
}

}  // namespace seq
}  // namespace fishing

using namespace fishing::seq;

extern "C" {

int fishing_embedding_forward(int32_t dtype, int32_t index_bytes, int64_t n, int64_t vocab, int64_t dim, const void* table, int64_t table_stride, const void* token,
                              float scale, void* out, fishing_stream_t stream) {
    if (int rc = embedding_check(dtype, index_bytes, n, vocab, dim)) return rc;
    if (table_stride < dim) return FISHING_ERR_SIZE;
    if (n == 0) return FISHING_OK;
    if (!table || !token || !out) return FISHING_ERR_NULL;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == FISHING_DTYPE_F32)
        return index_bytes == 4 ? embedding_forward<float, int32_t>(n, vocab, dim, (const float*)table, table_stride, (const int32_t*)token, scale, (float*)out, st)
                                : embedding_forward<float, int64_t>(n, vocab, dim, (const float*)table, table_stride, (const int64_t*)token, scale, (float*)out, st);
    return index_bytes == 4 ? embedding_forward<bf16, int32_t>(n, vocab, dim, (const bf16*)table, table_stride, (const int32_t*)token, scale, (bf16*)out, st)
                            : embedding_forward<bf16, int64_t>(n, vocab, dim, (const bf16*)table, table_stride, (const int64_t*)token, scale, (bf16*)out, st);
}

int64_t fishing_embedding_workspace(int32_t dtype, int64_t n, int64_t vocab, int64_t dim) {
    if (int rc = embedding_check(dtype, 4, n, vocab, dim)) return rc;
    return embedding_work(sort_plan(n, vocab, row_lanes(dtype, dim)), n, vocab, dim, nullptr).bytes;
}

int fishing_embedding_backward(int32_t dtype, int32_t index_bytes, int64_t n, int64_t vocab, int64_t dim, const void* dout, int64_t dout_stride, const void* token,
                               float scale, void* dtable, void* workspace, int64_t workspace_bytes, fishing_stream_t stream) {
    if (int rc = embedding_check(dtype, index_bytes, n, vocab, dim)) return rc;
    if (n > 0 && dout_stride < dim) return FISHING_ERR_SIZE;
    if (!dtable || !workspace || (n > 0 && (!dout || !token))) return FISHING_ERR_NULL;
    if (!aligned16(workspace)) return FISHING_ERR_ALIGN;
    if (workspace_bytes < fishing_embedding_workspace(dtype, n, vocab, dim)) return FISHING_ERR_SIZE;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == FISHING_DTYPE_F32)
        return index_bytes == 4 ? embedding_backward<float, int32_t>(n, vocab, dim, (const float*)dout, dout_stride, (const int32_t*)token, scale, (float*)dtable, workspace, st)
                                : embedding_backward<float, int64_t>(n, vocab, dim, (const float*)dout, dout_stride, (const int64_t*)token, scale, (float*)dtable, workspace, st);
    return index_bytes == 4 ? embedding_backward<bf16, int32_t>(n, vocab, dim, (const bf16*)dout, dout_stride, (const int32_t*)token, scale, (bf16*)dtable, workspace, st)
                            : embedding_backward<bf16, int64_t>(n, vocab, dim, (const bf16*)dout, dout_stride, (const int64_t*)token, scale, (bf16*)dtable, workspace, st);
}

}  // extern "C"
