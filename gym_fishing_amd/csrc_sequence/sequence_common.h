// sequence_common.h -- what the sequence operators' kernels share: element types, 16-byte accesses, the matrix-core tile
// wrappers of gfx950 and the launch helper.  The operators serve an agent that remembers its episode: token embedding
// (sequence_embedding.hip), linear attention with a decay per head (sequence_attention.hip), softmax cross entropy over the
// quota levels (sequence_loss.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include <tuple>

#include "../../include/fishing_hip.h"

namespace fishing {
namespace seq {

typedef __bf16 bf16;
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(bf16 x) { return (float)x; }
// round to nearest even (v_cvt_pk_bf16_f32): the one rounding of an output's last step
template <typename T>
__device__ __forceinline__ T from_f32(float x) { return (T)x; }

// N elements that move as one access (16 bytes for the vector forms, one element for the others)
template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
    T e[N];
};

template <typename T>
__host__ __device__ constexpr int vec_of() { return 16 / (int)sizeof(T); }

static inline bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }
__host__ __device__ inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
static inline int64_t round_up(int64_t a, int64_t b) { return ceil_div(a, b) * b; }

// This launch's own status, as hipLaunchKernel returns it
template <typename... P, typename... A>
inline int launch_lds(void (*kernel)(P...), dim3 grid, dim3 block, size_t lds, hipStream_t stream, A&&... args) {
    std::tuple<P...> packed{static_cast<P>(args)...};
    return std::apply(
        [&](auto&... a) {
            void* argv[] = {(void*)&a...};
            return (int)hipLaunchKernel((const void*)kernel, grid, block, argv, lds, stream);
        },
        packed);
}
template <typename... P, typename... A>
inline int launch(void (*kernel)(P...), dim3 grid, dim3 block, hipStream_t stream, A&&... args) {
    return launch_lds(kernel, grid, block, 0, stream, args...);
}

// Workspace carving: 256-byte aligned blocks in the caller's buffer
struct Carve {
    char* base;
    int64_t used = 0;
    explicit Carve(void* p) : base((char*)p) {}
    template <typename T>
    T* take(int64_t count) {
        T* p = (T*)(base + used);
        used = round_up(used + count * (int64_t)sizeof(T), 256);
        return p;
    }
};

// A value that is the same in every lane, into scalar registers: what a run-time division yields is in vector registers, and so
// would be every address made of it
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t uniform(int64_t x) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)x), hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)((uint64_t)x >> 32));
    return (int64_t)((uint64_t)hi << 32 | lo);
}

// Workgroups are dealt round-robin over the 8 XCDs, each with its own L2: hand each XCD a contiguous run
__device__ __forceinline__ int64_t xcd_run(int64_t id, int64_t count) {
    const int64_t per = count / 8, rest = count % 8, x = id % 8, at = id / 8;
    return x * per + (x < rest ? x : rest) + at;
}

}  // namespace seq
}  // namespace fishing
