// sequence_attention.hip -- linear attention with a decay for each head: over whole episodes with its gradient, and for the one
// step an env batch has just taken.
//
//   S_t = a_t S_{t-1} + k_t v_t^T        a_t = exp(log_decay[h]), or 0 where an episode starts at t
//   o_t = scale * q_t S_t
//
// and with R the gradient of the state behind step t, R_t = scale * q_t do_t^T + a_{t+1} R_{t+1} (R_{T-1} also takes the final state's):
//   dq_t = scale * S_t do_t      dk_t = R_t v_t      dv_t = R_t^T k_t      dS_{-1} = a_0 R_0
// so every gradient is the same recurrence with the roles of its operands exchanged, dk and dv backwards in time.
#include "sequence_walk.h"

namespace fishing {
namespace seq {

// ---- the single step: a wave owns one (env, head); its state goes through registers once, eight 16-byte loads a lane in flight.
// Bound by the state's two trips: 65536 envs, 4 heads of 32 x 32: 374 us a call back to back, 408 on average in a kernel trace (372 at
// best): 5.6 - 6.1 TB/s.  64 envs: 5 us of the call's 15, which are the host's ----
template <typename T, int V>
__global__ void __launch_bounds__(256) step_kernel_recurrent(Strided q, Strided k, Strided v, const float* log_decay, const uint8_t* starts, int64_t starts_stride,
                                                             const float* state, float* state_out, T* out, int64_t out_batch, int64_t out_head, int64_t pairs,
                                                             int32_t heads, int32_t dk, int32_t dv, float scale) {
    constexpr int U = 8;
    __shared__ float qk[4][2][kMaxHeadDim];
    __shared__ float part[4][64][V];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t pair = (int64_t)blockIdx.x * 4 + wave;
    const bool live = pair < pairs;
    const int64_t n = live ? pair / heads : 0;
    const int h = live ? (int)(pair - n * heads) : 0;
    const T* qp = (const T*)q.p + n * q.batch + h * q.head;
    const T* kp = (const T*)k.p + n * k.batch + h * k.head;
    const T* vp = (const T*)v.p + n * v.batch + h * v.head;
    if (live) {
        for (int i = lane; i < dk; i += 64) {
            qk[wave][0][i] = to_f32(qp[i]) * scale;
            qk[wave][1][i] = to_f32(kp[i]);
        }
    }
    __syncthreads();
    const float a = expf(log_decay_of(log_decay, h));
    const bool keep = !(starts && live && starts[n * starts_stride]) && a != 0.0f;       // (a decay of zero drops NaN too, as over whole episodes)
    const int cols = dv / V, wide = cols < 64 ? cols : 64, rows = 64 / wide;
    const int r = lane / wide, c0 = lane - r * wide;
    const float* from = state + pair * (int64_t)dk * dv;
    float* to = state_out + pair * (int64_t)dk * dv;
    for (int cb = 0; cb < cols; cb += 64) {
        const int c = cb + c0;
        const bool mine = live && r < rows && c < cols;
        float acc[V], vv[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            acc[e] = 0.0f;
            vv[e] = mine ? to_f32(vp[c * V + e]) : 0.0f;
        }
        if (mine) {
            for (int i0 = r; i0 < dk; i0 += rows * U) {
                Pack<float, V> s[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int i = i0 + u * rows;
                    if (i < dk && keep) s[u] = *(const Pack<float, V>*)(from + (int64_t)i * dv + c * V);
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int i = i0 + u * rows;
                    if (i < dk) {
                        const float qi = qk[wave][0][i], ki = qk[wave][1][i];
#pragma unroll
                        for (int e = 0; e < V; ++e) {
                            const float x = (keep ? a * s[u].e[e] : 0.0f) + ki * vv[e];
                            s[u].e[e] = x;
                            acc[e] += qi * x;
                        }
                        *(Pack<float, V>*)(to + (int64_t)i * dv + c * V) = s[u];
                    }
                }
            }
        }
#pragma unroll
        for (int e = 0; e < V; ++e) part[wave][lane][e] = acc[e];
        __syncthreads();
        if (mine && r == 0) {
            T* o = out + n * out_batch + h * out_head + c * V;
            for (int x = 1; x < rows; ++x) {
#pragma unroll
                for (int e = 0; e < V; ++e) acc[e] += part[wave][x * wide + c0][e];
            }
#pragma unroll
            for (int e = 0; e < V; ++e) o[e] = from_f32<T>(acc[e]);
        }
        __syncthreads();
    }
}

static int attention_check(const FishingDecayAttention* a, bool one_step) {
    if (!a) return FISHING_ERR_NULL;
    if (a->dtype != FISHING_DTYPE_F32 && a->dtype != FISHING_DTYPE_BF16) return FISHING_ERR_UNSUPPORTED;
    if (a->batch < 0 || a->steps < 0 || a->heads < 1 || a->dk < 1 || a->dk > kMaxHeadDim || a->dv < 1 || a->dv > kMaxHeadDim) return FISHING_ERR_SIZE;
    if (a->heads > kMaxHeads || a->batch > 0x7fffffff / a->heads) return FISHING_ERR_SIZE;
    if (a->batch == 0) return FISHING_OK;
    if (!a->log_decay) return FISHING_ERR_NULL;
    if ((one_step || a->steps > 0) && (!a->q || !a->k || !a->v)) return FISHING_ERR_NULL;
    return FISHING_OK;
}

static Strided strided(const void* p, const int64_t* s) { return Strided{p, s[0], s[1], s[2]}; }

template <typename T>
static int attention_step(const FishingDecayAttention* a, hipStream_t stream) {
    const int64_t block = batch_block(a->batch, a->heads), state = (int64_t)a->heads * a->dk * a->dv;
    auto go = [&](auto kernel) {
        int rc = 0;
        for (int64_t n = 0; n < a->batch && !rc; n += block) {
            const int64_t pairs = (a->batch - n < block ? a->batch - n : block) * a->heads;
            auto from = [&](const void* p, const int64_t* s) { return strided((const T*)p + n * s[0], s); };
            rc = launch(kernel, dim3((unsigned)ceil_div(pairs, 4)), dim3(256), stream, from(a->q, a->q_stride), from(a->k, a->k_stride), from(a->v, a->v_stride), a->log_decay,
                        a->starts ? a->starts + n * a->starts_stride[0] : nullptr, a->starts_stride[0], a->state + n * state, a->state_out + n * state,
                        (T*)a->out + n * a->out_stride[0], a->out_stride[0], a->out_stride[2], pairs, a->heads, a->dk, a->dv, (float)a->scale);
        }
        return rc;
    };
    if (a->dv % 4 == 0 && aligned16(a->state) && aligned16(a->state_out)) return go(step_kernel_recurrent<T, 4>);
    return go(step_kernel_recurrent<T, 1>);
}

extern template int walk<float, true>(const FishingDecayAttention*, Strided, Strided, Strided, const float*, float*, Strided, int, int, bool, bool, double, double, Shared*, void*, hipStream_t);
extern template int walk<bf16, true>(const FishingDecayAttention*, Strided, Strided, Strided, const float*, float*, Strided, int, int, bool, bool, double, double, Shared*, void*, hipStream_t);

template <typename T>
static int attention_forward(const FishingDecayAttention* a, void* work, hipStream_t stream) {
    return walk<T, false>(a, strided(a->q, a->q_stride), strided(a->k, a->k_stride), strided(a->v, a->v_stride), a->state, a->state_out,
                               strided((const void*)a->out, a->out_stride), a->dk, a->dv, false, true, a->scale, 1.0, nullptr, work, stream);
}

template <typename T>
static int attention_backward(const FishingDecayAttention* a, void* work, hipStream_t stream) {
    const Strided q = strided(a->q, a->q_stride), k = strided(a->k, a->k_stride), v = strided(a->v, a->v_stride), g = strided(a->dout, a->dout_stride);
    // dq: read with do the state that (v, k) build;  dk, dv: read with v, k the state's gradient that (do, q), (q, do) build backwards,
    // in segments from the same states
    Shared both;
    both.exact = a->dstate != nullptr;
    int rc = walk<T, false>(a, g, v, k, a->state, nullptr, strided((const void*)a->dq, a->dq_stride), a->dv, a->dk, true, false, a->scale, 1.0, nullptr, work, stream);
    if (!rc) rc = walk<T, true>(a, v, g, q, a->dstate_out, nullptr, strided((const void*)a->dk_out, a->dk_stride), a->dv, a->dk, true, false, 1.0, a->scale, &both, work, stream);
    if (!rc)
        rc = walk<T, true>(a, k, q, g, a->dstate_out, a->dstate, strided((const void*)a->dv_out, a->dv_stride), a->dk, a->dv, false, a->dstate != nullptr, 1.0, a->scale, &both,
                           work, stream);
    return rc;
}

}  // namespace seq
}  // namespace fishing

using namespace fishing::seq;

extern "C" {

int fishing_decay_attention_step(const FishingDecayAttention* a, fishing_stream_t stream) {
    if (int rc = attention_check(a, true)) return rc;
    if (a->batch == 0) return FISHING_OK;
    if (!a->state || !a->state_out || !a->out) return FISHING_ERR_NULL;
    return a->dtype == FISHING_DTYPE_F32 ? attention_step<float>(a, (hipStream_t)stream) : attention_step<bf16>(a, (hipStream_t)stream);
}

int64_t fishing_decay_attention_workspace(const FishingDecayAttention* a, int32_t backward) {
    if (int rc = attention_check(a, false)) return rc;
    // the largest of its walks, which run one after the other, whichever way their rows are read; dk's and dv's share dk's states
    const int64_t pairs = batch_block(a->batch, a->heads) * a->heads;
    int64_t most = 0, flags = 0;
    for (int back = 0; back <= (backward ? 1 : 0); ++back)
        for (int wide = 0; wide < 2; ++wide) {
            const int rows = back ? a->dv : a->dk, cols = back ? a->dk : a->dv;
            const WalkPlan p = walk_plan(a->dtype, pairs, a->steps, rows, cols, wide != 0);
            const int64_t b = walk_work(p, pairs, cols, nullptr, nullptr).bytes, f = round_up(pairs * ceil_div(a->dv, 32) * p.segs * (int64_t)sizeof(uint32_t), 256);
            most = b > most ? b : most;
            if (back && p.segs > 1) flags = f > flags ? f : flags;
        }
    most += flags;
    return most;
}

int fishing_decay_attention_forward(const FishingDecayAttention* a, void* workspace, int64_t workspace_bytes, fishing_stream_t stream) {
    if (int rc = attention_check(a, false)) return rc;
    if (a->batch == 0) return FISHING_OK;
    if ((a->steps > 0 && !a->out) || !workspace) return FISHING_ERR_NULL;
    if (!aligned16(workspace)) return FISHING_ERR_ALIGN;
    if (workspace_bytes < fishing_decay_attention_workspace(a, 0)) return FISHING_ERR_SIZE;
    return a->dtype == FISHING_DTYPE_F32 ? attention_forward<float>(a, workspace, (hipStream_t)stream) : attention_forward<bf16>(a, workspace, (hipStream_t)stream);
}

int fishing_decay_attention_backward(const FishingDecayAttention* a, void* workspace, int64_t workspace_bytes, fishing_stream_t stream) {
    if (int rc = attention_check(a, false)) return rc;
    if (a->batch == 0) return FISHING_OK;
    if ((a->steps > 0 && (!a->dout || !a->dq || !a->dk_out || !a->dv_out)) || !workspace) return FISHING_ERR_NULL;
    if (!aligned16(workspace)) return FISHING_ERR_ALIGN;
    if (workspace_bytes < fishing_decay_attention_workspace(a, 1)) return FISHING_ERR_SIZE;
    return a->dtype == FISHING_DTYPE_F32 ? attention_backward<float>(a, workspace, (hipStream_t)stream) : attention_backward<bf16>(a, workspace, (hipStream_t)stream);
}

}  // extern "C"
