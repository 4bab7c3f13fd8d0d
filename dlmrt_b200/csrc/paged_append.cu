// New tokens enter the paged cache: per-head norm, rotation, and the store of keys and values into their slots, with the
// rotated queries written on the way (dlmrt/ops/triton/core.py: QK-norm + RoPE + KV write, one launch there too).
//
//   y = x * rsqrt(mean(x^2) + eps) * weight          over a head, where a weight is given
//   (a, b) -> (a cos - b sin, b cos + a sin)          on the first `rotated` elements, pairs i, i + rotated / 2 or 2i, 2i + 1
//
// Everything is FP32 between the load and the one rounding at the store. A block takes one token. A head row is spread over
// head_dim / 8 lanes, 16 bytes each: the partner of a rotated element sits in another lane of the same group (one shuffle per
// element) or, for neighbouring pairs, in the same lane, and a lane's cosines and sines are the same for all heads. Bound by
// HBM for prompts: each lane has up to four heads' loads on the way at once, before the token's position and slot are known,
// and registers are held to five blocks an SM, although 16-bit caches then spill 184 bytes a thread (8189 tokens of 32 head rows of
// 256: 98 us with one row a lane, 65 with four at three blocks an SM, 53.5 at five). FP8 caches, at four, do not spill.
#include <climits>

#include "../../include/dlmrt_b200.h"
#include "mma.cuh"
#include "serving.cuh"

namespace dlm {

namespace {

constexpr int kAppendMostThreads = 256;
constexpr int kHeadsAtOnce = 4;  // head rows that a lane has on the way

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

// Apart from the kernel, whose registers are few.
__device__ __noinline__ void report_token(int* status, int token, bool bad_slot, long long slot, int page_shift, int pos) {
    const long long page = slot >> page_shift;
    if (bad_slot)
        report_index(status, token, kIndexSlot, page > INT_MAX ? INT_MAX : static_cast<int>(page),
                     static_cast<int>(slot & ((1ll << page_shift) - 1)));
    else
        report_index(status, token, kIndexPosition, pos);
}

}  // namespace

template <typename T, int D, bool kCodes>
__global__ void __launch_bounds__(kAppendMostThreads, kCodes ? 4 : 5) append_kernel(const __grid_constant__ DlmAppend p, int page_shift) {
    constexpr int kLanes = D / 8;  // lanes of one head row
    const int lane = static_cast<int>(threadIdx.x) % kLanes, group = static_cast<int>(threadIdx.x) / kLanes;
    const int groups = static_cast<int>(blockDim.x) / kLanes;
    const int q_heads = p.q != nullptr ? p.q_heads : 0, heads = p.cache.heads;
    const int rows = q_heads + 2 * heads;  // queries, keys, values
    const long long token = blockIdx.x;
    pdl_wait();
    pdl_launch_dependents();
    const long long slot = p.slots[token];
    const int pos = p.rotated ? p.positions[token] : 0;
    const T* q = static_cast<const T*>(p.q) + token * p.q_strides[0] + lane * 8;
    const T* k = static_cast<const T*>(p.k) + token * p.k_strides[0] + lane * 8;
    const T* v = static_cast<const T*>(p.v) + token * p.v_strides[0] + lane * 8;
    auto load = [&](int row) {
        const T* src = row < q_heads           ? q + row * p.q_strides[1]
                       : row < q_heads + heads ? k + (row - q_heads) * p.k_strides[1]
                                               : v + (row - q_heads - heads) * p.v_strides[1];
        return *reinterpret_cast<const uint4*>(src);
    };
    // The same number of passes for every group: all lanes of a warp take part in the shuffles.
    for (int base = group; base - group < rows; base += groups * kHeadsAtOnce) {
        uint4 raw[kHeadsAtOnce];
#pragma unroll
        for (int i = 0; i < kHeadsAtOnce; ++i) {
            const int row = base + i * groups;
            raw[i] = row < rows ? load(row) : make_uint4(0, 0, 0, 0);
        }
        const bool bad_slot = slot >= static_cast<long long>(p.cache.pages) << page_shift;
        const bool bad_pos = p.rotated && (pos < 0 || pos >= p.table_rows);
        if (bad_slot || bad_pos) {  // nothing of this token is written
            if (threadIdx.x == 0) report_token(p.cache.status, static_cast<int>(token), bad_slot, slot, page_shift, pos);
            return;
        }
        // This lane's cosines and sines; partner: the lane that holds the other halves of its pairs.
        float cs[8], sn[8];
        const int half = p.rotated / 2, step = half / 8;
        const bool turned = lane * 8 < p.rotated, first = lane < step;
        const int partner = (static_cast<int>(threadIdx.x) & 31) + (!turned || p.interleaved ? 0 : first ? step : -step);
        if (turned) {
            const float* row = p.table + static_cast<long long>(pos) * p.rotated;
            if (p.interleaved) {
                *reinterpret_cast<float4*>(cs) = *reinterpret_cast<const float4*>(row + lane * 4);
                *reinterpret_cast<float4*>(sn) = *reinterpret_cast<const float4*>(row + half + lane * 4);
            } else {
                const float* at = row + (first ? lane : lane - step) * 8;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    *reinterpret_cast<float4*>(cs + 4 * i) = *reinterpret_cast<const float4*>(at + 4 * i);
                    *reinterpret_cast<float4*>(sn + 4 * i) = *reinterpret_cast<const float4*>(at + half + 4 * i);
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) sn[i] = first ? -sn[i] : sn[i];  // x * cos + partner * sn, for both halves
            }
        }
#pragma unroll
        for (int i = 0; i < kHeadsAtOnce; ++i) {
            const int row = base + i * groups;
            const bool is_q = row < q_heads, is_v = row >= q_heads + heads;
            const int head = is_q ? row : is_v ? row - q_heads - heads : row - q_heads;
            const T* norm = static_cast<const T*>(is_v ? nullptr : is_q ? p.q_norm : p.k_norm);
            float x[8];
            unpack8<T>(raw[i], x);
            if (p.q_norm != nullptr || p.k_norm != nullptr) {
                float sum = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) sum += x[j] * x[j];
#pragma unroll
                for (int o = kLanes / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
                if (norm != nullptr) {
                    const float r = rsqrtf(sum * (1.f / D) + p.eps);
                    float w[8];
                    unpack8<T>(*reinterpret_cast<const uint4*>(norm + lane * 8), w);
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[j] = x[j] * r * w[j];
                }
            }
            if (p.rotated && p.interleaved) {
                if (turned && !is_v) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float a = x[2 * j], b = x[2 * j + 1];
                        x[2 * j] = a * cs[j] - b * sn[j];
                        x[2 * j + 1] = b * cs[j] + a * sn[j];
                    }
                }
            } else if (p.rotated) {
                float other[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) other[j] = __shfl_sync(0xFFFFFFFFu, x[j], partner);
                if (turned && !is_v) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[j] = x[j] * cs[j] + other[j] * sn[j];
                }
            }
            if (row >= rows || (slot < 0 && !is_q)) continue;
            const bool as_is = norm == nullptr && (is_v || !p.rotated);  // a copy keeps its bits, those of a NaN among them
            if (is_q) {
                T* dst = static_cast<T*>(p.q_out) + token * p.out_strides[0] + head * p.out_strides[1] + lane * 8;
                *reinterpret_cast<uint4*>(dst) = as_is ? raw[i] : pack8<T>(x);
                continue;
            }
            const int64_t* st = is_v ? p.cache.v_strides : p.cache.k_strides;
            const long long page = slot >> page_shift, within = slot & ((1ll << page_shift) - 1);
            const long long at = page * st[0] + head * st[1] + within * st[2] + lane * 8;
            void* pool = is_v ? p.cache.values : p.cache.keys;
            if constexpr (kCodes) {
                const float scale = (is_v ? p.cache.v_scale : p.cache.k_scale)[head];
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = x[j] / scale;
                *reinterpret_cast<uint2*>(static_cast<uint8_t*>(pool) + at) =
                    make_uint2(e4m3x4(x[0], x[1], x[2], x[3]), e4m3x4(x[4], x[5], x[6], x[7]));
            } else {
                *reinterpret_cast<uint4*>(static_cast<T*>(pool) + at) = as_is ? raw[i] : pack8<T>(x);
            }
        }
    }
}

template <typename T, int D>
static int launch_append_d(const DlmAppend& p, int page_shift, const LaunchOpts& o) {
    const int rows = (p.q != nullptr ? p.q_heads : 0) + 2 * p.cache.heads;
    const int lanes = (rows + kHeadsAtOnce - 1) / kHeadsAtOnce * (D / 8);
    const int threads = lanes >= kAppendMostThreads ? kAppendMostThreads : (lanes + 31) / 32 * 32;
    void* args[] = {const_cast<DlmAppend*>(&p), &page_shift};
    return p.cache.type == DLM_E4M3 ? launch_kernel<append_kernel<T, D, true>>(dim3(p.n), dim3(threads), 0, args, o)
                                    : launch_kernel<append_kernel<T, D, false>>(dim3(p.n), dim3(threads), 0, args, o);
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
