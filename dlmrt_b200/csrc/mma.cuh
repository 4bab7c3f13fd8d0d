// Warp-level building blocks of the kernels whose rows are too few for a 128-row tensor-memory tile: mma.sync on 16-bit
// operands with FP32 accumulation, ldmatrix and movmatrix, FP8 widening; and the launch of one kernel.
#pragma once

#include <cuda_fp16.h>

#include <type_traits>

#include "kernels.cuh"

namespace dlm {

// D[16, 8] += A[16, 16] * B[16, 8]. With g = lane / 4, t = lane % 4: a0 holds A[g][2t, 2t + 1], a1 row g + 8, a2 columns
// + 8, a3 both; b0 holds B[2t, 2t + 1][g], b1 rows + 8; d0, d1 are D[g][2t, 2t + 1], d2, d3 row g + 8.
template <typename T>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __half>::value) {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    } else {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
}

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t smem) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(smem)
                 : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t smem) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(smem)
                 : "memory");
}

// The 8x8 matrix whose row lane / 4 has this lane's two 16-bit elements in columns 2 (lane % 4) and the next, transposed.
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
    uint32_t out;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(out) : "r"(v));
    return out;
}

// Two E4M3 codes (low byte first) as two halves: exact.
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t codes) {
    uint32_t h2;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"(static_cast<uint16_t>(codes)));
    return h2;
}

// Four values as E4M3 codes, the first in the low byte: to nearest, at most the largest code in magnitude, NaN stays NaN.
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    return static_cast<uint32_t>(lo) | static_cast<uint32_t>(hi) << 16;
}

template <typename T>
__device__ __forceinline__ float2 widen2(uint32_t v) {
    if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&v));
    else return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
}
template <typename T>
__device__ __forceinline__ uint32_t narrow2(float x, float y) {
    uint32_t out;
    if constexpr (std::is_same<T, __half>::value) *reinterpret_cast<__half2*>(&out) = __floats2half2_rn(x, y);
    else *reinterpret_cast<__nv_bfloat162*>(&out) = __floats2bfloat162_rn(x, y);
    return out;
}

// Two halves rounded towards zero; zero for what is below.
__device__ __forceinline__ uint32_t narrow2_down_to_zero(float x, float y) {
    uint32_t out;
    asm("cvt.rz.relu.f16x2.f32 %0, %1, %2;" : "=r"(out) : "f"(y), "f"(x));
    return out;
}

__device__ __forceinline__ float exp2_approx(float x) {  // relative error about 2^-22, exp2(-inf) = 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Launches `Kernel`; where it takes more dynamic shared memory than any kernel may, its limit is raised once per device, to
// `smem` (then the same at every call).
template <auto Kernel>
int launch_kernel(dim3 grid, dim3 block, int smem, void** args, const LaunchOpts& o, int cluster = 1) {
    const void* kernel = reinterpret_cast<const void*>(Kernel);
    cudaLaunchConfig_t config{};
    config.gridDim = grid;
    config.blockDim = block;
    config.dynamicSmemBytes = static_cast<size_t>(smem);
    config.stream = o.stream;
    cudaLaunchAttribute attrs[2]{};
    int n = 0;
    if (o.pdl) {
        attrs[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attrs[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 1) {
        attrs[n].id = cudaLaunchAttributeClusterDimension;
        attrs[n].val.clusterDim.x = static_cast<unsigned>(cluster);
        attrs[n].val.clusterDim.y = attrs[n].val.clusterDim.z = 1;
        ++n;
    }
    config.attrs = attrs;
    config.numAttrs = static_cast<unsigned>(n);
    cudaError_t err = cudaSuccess;
    if (smem > 40 * 1024) {
        static bool raised[64] = {};
        int dev = 0;
        err = cudaGetDevice(&dev);
        if (err == cudaSuccess && (dev >= 64 || !raised[dev])) {
            err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
            if (dev < 64) raised[dev] = err == cudaSuccess;
        }
    }
    if (err == cudaSuccess) err = cudaLaunchKernelExC(&config, kernel, args);
    if (err != cudaSuccess) {
        g_last_cuda_error = static_cast<int>(err);
        (void)cudaGetLastError();
        return -6;
    }
    ++g_launches;
    return 0;
}

}  // namespace dlm
