// New tokens enter the paged cache: per-head norm, rotation, and the store of keys and values into their slots, with the
// rotated queries written on the way (dlmrt/ops/triton/core.py: QK-norm + RoPE + KV write, one launch there too).
//
//   y = x * rsqrt(mean(x^2) + eps) * weight          over a head, where a weight is given
//   (a, b) -> (a cos - b sin, b cos + a sin)          on the first `rotated` elements, pairs i, i + rotated / 2 or 2i, 2i + 1
//
// Everything is FP32 between the load and the one rounding at the store. A head row is spread over head_dim / 8 lanes, 16
// bytes each: the partner of a rotated element sits in another lane of the same group (one shuffle per element) or, for
// neighbouring pairs, in the same lane.
#include "../../include/dlmrt_b200.h"
#include "mma.cuh"
#include "serving.cuh"

namespace dlm {

namespace {

constexpr int kAppendThreads = 256;

template <typename T>
__device__ __forceinline__ void unpack8(const uint4& raw, float (&v)[8]) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = widen2<T>(w[i]);
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
    }
}

template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
    return make_uint4(narrow2<T>(v[0], v[1]), narrow2<T>(v[2], v[3]), narrow2<T>(v[4], v[5]), narrow2<T>(v[6], v[7]));
}

__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {  // saturating, NaN stays NaN
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    return static_cast<uint32_t>(lo) | static_cast<uint32_t>(hi) << 16;
}

}  // namespace

template <typename T, int D, bool kCodes>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const __grid_constant__ DlmAppend p, int page_shift) {
    constexpr int kLanes = D / 8;                       // lanes of one head row
    constexpr int kRows = kAppendThreads / kLanes;      // head rows of a block
    const int lane = static_cast<int>(threadIdx.x) % kLanes;
    const int q_heads = p.q != nullptr ? p.q_heads : 0, heads = p.cache.heads;
    const int per_token = q_heads + 2 * heads;
    const long long item = static_cast<long long>(blockIdx.x) * kRows + static_cast<int>(threadIdx.x) / kLanes;
    const long long token = item / per_token;
    const int which = static_cast<int>(item - token * per_token);
    const bool is_q = which < q_heads, is_v = which >= q_heads + heads;
    const int head = is_q ? which : is_v ? which - q_heads - heads : which - q_heads;
    pdl_wait();
    pdl_launch_dependents();
    bool live = token < p.n;
    int pos = 0;
    long long slot = -1;
    if (live) {
        slot = p.slots[token];
        if (p.rotated) pos = p.positions[token];
        const bool bad_slot = slot >= static_cast<long long>(p.cache.pages) << page_shift;
        const bool bad_pos = p.rotated && (pos < 0 || pos >= p.table_rows);
        if (bad_slot || bad_pos) {
            if (which == 0 && lane == 0)
                report_index(p.cache.status, static_cast<int>(token), bad_slot ? kIndexSlot : kIndexPosition,
                             bad_slot ? static_cast<int>(slot >> page_shift) : pos);
            live = false;
        }
        if (slot < 0 && !is_q) live = false;
    }
    float v[8] = {};
    uint4 raw = make_uint4(0, 0, 0, 0);
    if (live) {
        const T* src = is_q ? static_cast<const T*>(p.q) + token * p.q_strides[0] + head * p.q_strides[1]
                     : is_v ? static_cast<const T*>(p.v) + token * p.v_strides[0] + head * p.v_strides[1]
                            : static_cast<const T*>(p.k) + token * p.k_strides[0] + head * p.k_strides[1];
        raw = *reinterpret_cast<const uint4*>(src + lane * 8);
        unpack8<T>(raw, v);
    }
    // The rows of one warp may be queries, keys and values: every lane takes part in the shuffles, whoever uses them.
    const T* norm = static_cast<const T*>(is_v ? nullptr : is_q ? p.q_norm : p.k_norm);
    if (p.q_norm != nullptr || p.k_norm != nullptr) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += v[i] * v[i];
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
        if (norm != nullptr) {
            const float r = rsqrtf(sum * (1.f / D) + p.eps);
            float w[8];
            unpack8<T>(*reinterpret_cast<const uint4*>(norm + lane * 8), w);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = v[i] * r * w[i];
        }
    }
    if (p.rotated) {
        const int half = p.rotated / 2;
        const bool turned = live && !is_v && lane * 8 < p.rotated;
        const float* row = p.table + static_cast<long long>(turned ? pos : 0) * p.rotated;
        if (p.interleaved) {
            if (turned) {
                const float4 c = *reinterpret_cast<const float4*>(row + lane * 4);
                const float4 s = *reinterpret_cast<const float4*>(row + half + lane * 4);
                const float cs[4] = {c.x, c.y, c.z, c.w}, sn[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float a = v[2 * i], b = v[2 * i + 1];
                    v[2 * i] = a * cs[i] - b * sn[i];
                    v[2 * i + 1] = b * cs[i] + a * sn[i];
                }
            }
        } else {
            const int step = half / 8;  // lanes between a pair's elements
            const bool first = lane < step;
            const int base = (static_cast<int>(threadIdx.x) & 31) - lane;
            const int from = base + (lane * 8 < p.rotated ? (first ? lane + step : lane - step) : lane);
            float other[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) other[i] = __shfl_sync(0xFFFFFFFFu, v[i], from);
            if (turned) {
                const float* at = row + (first ? lane : lane - step) * 8;
                float cs[8], sn[8];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    *reinterpret_cast<float4*>(cs + 4 * i) = *reinterpret_cast<const float4*>(at + 4 * i);
                    *reinterpret_cast<float4*>(sn + 4 * i) = *reinterpret_cast<const float4*>(at + half + 4 * i);
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = first ? v[i] * cs[i] - other[i] * sn[i] : v[i] * cs[i] + other[i] * sn[i];
            }
        }
    }
    if (!live) return;
    const bool as_is = norm == nullptr && (is_v || !p.rotated);  // a copy keeps its bits, those of a NaN among them
    if (is_q) {
        T* dst = static_cast<T*>(p.q_out) + token * p.out_strides[0] + head * p.out_strides[1];
        *reinterpret_cast<uint4*>(dst + lane * 8) = as_is ? raw : pack8<T>(v);
        return;
    }
    const int64_t* st = is_v ? p.cache.v_strides : p.cache.k_strides;
    const long long page = slot >> page_shift, within = slot & ((1ll << page_shift) - 1);
    const long long at = page * st[0] + head * st[1] + within * st[2] + lane * 8;
    void* pool = is_v ? p.cache.values : p.cache.keys;
    if constexpr (kCodes) {
        const float scale = (is_v ? p.cache.v_scale : p.cache.k_scale)[head];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = v[i] / scale;
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(pool) + at) =
            make_uint2(e4m3x4(v[0], v[1], v[2], v[3]), e4m3x4(v[4], v[5], v[6], v[7]));
    } else {
        *reinterpret_cast<uint4*>(static_cast<T*>(pool) + at) = as_is ? raw : pack8<T>(v);
    }
}

template <typename T, int D>
static int launch_append_d(const DlmAppend& p, int page_shift, const LaunchOpts& o) {
    const long long items = static_cast<long long>(p.n) * ((p.q != nullptr ? p.q_heads : 0) + 2 * p.cache.heads);
    constexpr int kRows = kAppendThreads / (D / 8);
    void* args[] = {const_cast<DlmAppend*>(&p), &page_shift};
    const dim3 grid(static_cast<unsigned>((items + kRows - 1) / kRows));
    return p.cache.type == DLM_E4M3 ? launch_kernel<append_kernel<T, D, true>>(grid, dim3(kAppendThreads), 0, args, o)
                                    : launch_kernel<append_kernel<T, D, false>>(grid, dim3(kAppendThreads), 0, args, o);
}

int launch_append(const DlmAppend& p, int page_shift, const LaunchOpts& o) {
    auto by_dim = [&](auto t) {
        using T = decltype(t);
        switch (p.cache.head_dim) {
            case 64: return launch_append_d<T, 64>(p, page_shift, o);
            case 128: return launch_append_d<T, 128>(p, page_shift, o);
            default: return launch_append_d<T, 256>(p, page_shift, o);
        }
    };
    return p.type == DLM_F16 ? by_dim(__half{}) : by_dim(__nv_bfloat16{});
}

}  // namespace dlm
