// Shared by the latent-attention launchers: sizes, 16-bit types, the rotation of the position values, launch helper.
//
// A layer with latent attention keeps one row of 576 values per token for all of its heads: a latent of 512 that is key and
// value at once, and 64 rotated values that are key only.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "launch_common.h"

namespace vib3 {

extern std::atomic<int> g_use_pdl;   // vib3_config_set key 1

constexpr int kRank = 512;            // latent values of a row
constexpr int kRope = 64;             // position values of a row
constexpr int kLatentRow = kRank + kRope;
constexpr int kLatentMaxHeads = 128;
constexpr int kStatusBadPage = 1;     // VIB3_STATUS_MISSING_PAGE
constexpr int kStatusTimeout = 4;     // VIB3_STATUS_TIMEOUT

// The activation codes of the C ABI.
enum LatentDType : int { L_F32 = 0, L_F16 = 1, L_BF16 = 2 };

template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// Two floats as one 32-bit word of two T, `lo` in the low half.
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t v) {
    const T* t = reinterpret_cast<const T*>(&v);
    return make_float2(as_float(t[0]), as_float(t[1]));
}

// Cosine and sine of position * inv_freq.  The angle of a far position has no 32-bit form that keeps its fraction of a turn
// (at 200,000 the spacing of fp32 is 1/64): it is formed and reduced to [-pi, pi] in 64 bits and only then rounded.
__device__ __forceinline__ void rope_angle(int position, double inv_freq, float scale, float& c, float& s) {
    constexpr double kTurn = 6.283185307179586476925, kPerTurn = 0.15915494309189533577;
    double a = (double)position * inv_freq;
    a -= rint(a * kPerTurn) * kTurn;
    sincosf((float)a, &s, &c);
    c *= scale;
    s *= scale;
}

// Every latent kernel starts with pdl_enter(): nothing of its inputs is read before the predecessor in the stream has
// finished (its weights may be what the predecessor wrote), and the successor may start only after that, so that a launch
// that reads older data before its own wait still finds it complete.  What overlaps is the launch itself.
__device__ __forceinline__ void pdl_wait_only() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pdl_enter() {
    pdl_wait_only();
    pdl_release();
}

template <class K, class... Args>
int launch_latent(K kernel, dim3 grid, int threads, size_t smem, cudaStream_t st, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = g_use_pdl.load(std::memory_order_relaxed) ? 1 : 0;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
    if (e != cudaSuccess) (void)cudaGetLastError();   // reported by the return value, not by the next call
    return (int)e;
}

}  // namespace vib3
