// Shared by the tensor-core kernels of latent attention: barriers with bounded waits, tensor copies, tcgen05 operands and maps.
#pragma once
#include <cuda.h>

#include <type_traits>

#include "latent_common.cuh"

namespace vib3 {

int sm_count();

constexpr int kChunkBytes = 64 * 128;   // 64 rows of 64 values, 128-byte swizzle: the unit of the operands in shared memory

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint64_t* bar, unsigned count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_expect(uint64_t* bar, unsigned bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// Waits for the phase with this parity; gives up, with false, after about four seconds (a try comes back after some 4 us).
__device__ __forceinline__ bool bar_wait(uint64_t* bar, unsigned parity) {
    const uint32_t addr = smem_u32(bar);
    uint32_t ok = 0;
    for (unsigned it = 0; !ok && it < (1u << 20); ++it)
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(ok) : "r"(addr), "r"(parity) : "memory");
    return ok != 0;
}
// The same for a whole warp, whose lanes have to agree (they meet again in warp-wide instructions).
__device__ __forceinline__ bool bar_wait_warp(uint64_t* bar, unsigned parity) { return __all_sync(0xffffffffu, bar_wait(bar, parity)); }
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// One lane of the warp, the same one every time: behind elect.sync MMAs and tensor copies issue back to back.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void umma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// Shared-memory operands with 128-byte swizzle.  K-major: rows of 128 bytes, eight of them 1024 bytes.  MN-major: 64 values
// contiguous per key, eight keys 1024 bytes, the next 64 values a chunk further.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_k(uint32_t addr) { return ((addr & 0x3FFFF) >> 4) | (1u << 16); }
__device__ __forceinline__ uint32_t desc_mn(uint32_t addr) { return ((addr & 0x3FFFF) >> 4) | ((uint32_t)(kChunkBytes >> 4) << 16); }
// A value that is the same in all lanes, told to the compiler: an MMA takes its operands from uniform registers, and with
// operands that it had to move there one by one an MMA of this kernel cost 85 cycles instead of the pipe's 32 or 48.
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); }
// Operands by the low words of their descriptors (the address); the high words are constants.
__device__ __forceinline__ void umma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tmov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}"
                 ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "n"(kDescHigh) : "memory");
}
// The same with the first operand in tensor memory.
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tmov.b64 b, {%2, %5};\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "r"(b_lo), "r"(idesc), "r"(accumulate), "n"(kDescHigh) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// 32 lanes x 32 columns, a lane per thread.
__device__ __forceinline__ void tmem_ld_32x32(uint32_t taddr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(taddr) : "memory");
}

// Instruction descriptor: fp32 accumulator of m x n, both operands of type T, each with K or MN contiguous.
template <typename T>
constexpr uint32_t idesc(uint32_t m, uint32_t n, bool a_mn, bool b_mn) {
    const uint32_t format = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    return (1u << 4) | (format << 7) | (format << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) | (n / 8 << 17) | (m / 16 << 24);
}

typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                             const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeFn tensor_map_encoder() {
    static EncodeFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult r;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &r) != cudaSuccess) {
            p = nullptr;
            (void)cudaGetLastError();
        }
        return reinterpret_cast<EncodeFn>(p);
    }();
    return fn;
}

// Rows of `width` 16-bit values as x, ys rows y_stride apart as y, zs of those z_stride apart as z (strides in values); a copy takes 64 x
// box_y x box_z of them, with 128-byte swizzle.  Outside is read as zeros and not written.  False where the driver refuses it.
inline bool map_3d(CUtensorMap* m, int dtype, const void* base, long long width, long long ys, long long zs, long long y_stride, long long z_stride,
                   int box_y, int box_z) {
    const cuuint64_t dims[3] = {(cuuint64_t)width, (cuuint64_t)ys, (cuuint64_t)zs};
    const cuuint64_t strides[2] = {(cuuint64_t)y_stride * 2, (cuuint64_t)z_stride * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)box_y, (cuuint32_t)box_z}, one[3] = {1, 1, 1};
    return tensor_map_encoder()(m, dtype == L_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base),
                                dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Lets a kernel have `bytes` of dynamic shared memory: once per device and kernel.
template <auto kKernel>
int allow_smem(int bytes) {
    static std::atomic<unsigned long long> done{0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && (dev > 63 || !(done.load(std::memory_order_acquire) >> dev & 1))) {
        e = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e == cudaSuccess && dev <= 63) done.fetch_or(1ull << dev, std::memory_order_release);
    }
    if (e != cudaSuccess) (void)cudaGetLastError();
    return (int)e;
}

}  // namespace vib3
