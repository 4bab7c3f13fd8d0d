// Low-rank adapters of many requests beside a shared projection:
//
//   out[i] = base[i] + scale[id] * (x[i] A[id]^T) B[id]^T,   id = ids[i]
//
// Bound by reading the adapters' matrices once (rank * (k + n) * 2 bytes each) and, for the small sizes of a block of
// rows, by the chain of latencies between the two products. One launch does both: a cluster of eight CTAs takes up to 16
// rows of one adapter (the M of an mma.sync). Its CTAs split k for x A^T, add their FP32 partial sums through each other's
// shared memory in rank order (so the value never depends on timing), and split n for the second product, whose first
// operands are on their way before the exchange.
//
// Which rows form a cluster is read off `ids` by the cluster itself: a row leads if it is the 1st, 17th, 33rd ... of its
// adapter, and cluster c takes the c-th leader's adapter and that row's next fellows, up to 16. No sort, no host round trip,
// any order of ids. There are at most count + m / 16 leaders.
//
// 61 rows of 48 adapters, rank 16, k 2560, n 9728: 9.3 to 9.6 us (2.3 TB/s); 256 rows of 8 adapters, rank 64, k 9728, n 2560:
// 13.4 to 14.2 us.
#include <cooperative_groups.h>

#include "mma.cuh"
#include "serving.cuh"

namespace dlm {

namespace {

constexpr int kAdapterCtas = 8;
constexpr int kAdapterRows = 16;
constexpr int kMostRows = 256;

constexpr int kWarps = 8, kThreads = kWarps * 32;  // a thread for each row that a call may have
static_assert(kThreads == kMostRows, "a thread looks at one row's id");

// kTiles: n8 tiles of the first product's output, rank / 8 rounded up. CTAs of an SM: rank 16 with 48 adapters is 408 CTAs,
// in one wave at three an SM (12 us) but three waves at one (22 us, with 16 warps each).
template <int kTiles>
constexpr int adapter_ctas() {
    return kTiles <= 2 ? 3 : kTiles <= 8 ? 2 : 1;
}

template <int kTiles>
struct AdapterSmem {
    float part[kWarps][kAdapterRows][kTiles * 8 + 4];
    float sum[kAdapterRows][kTiles * 8];                    // this CTA's share of x A^T, read by the cluster
    uint32_t high[kAdapterRows][kTiles * 4 + 4];            // x A^T times the scale, BF16 pairs
    uint32_t low[kAdapterRows][kTiles * 4 + 4];             // what those leave over, BF16 pairs
    int ids[kMostRows];
    int2 kinds[kWarps][32];  // adapter, rows of it; behind the last one -1
    int kind_count[kWarps];
    int rows[kAdapterRows];
    uint32_t leads[kMostRows / 32];
    int lead, lead_before;
};

// A value as the sum of two BF16 ones. The high part is the nearest, or the largest below a finite value that would become
// infinite; of an infinity both parts are infinite (inf - inf would be NaN).
__device__ __forceinline__ float high_part(float v) {
    const float nearest = __bfloat162float(__float2bfloat16_rn(v));
    return isinf(nearest) && !isinf(v) ? __uint_as_float(__float_as_uint(v) & 0xFFFF0000u) : nearest;
}
__device__ __forceinline__ float low_part(float v, float high) { return isinf(v) ? v : v - high; }

}  // namespace

template <int kTiles>
__global__ void __launch_bounds__(kThreads, adapter_ctas<kTiles>()) adapters_kernel(const __grid_constant__ DlmAdapters p) {
    namespace cg = cooperative_groups;
    extern __shared__ __align__(16) uint8_t raw[];
    AdapterSmem<kTiles>& sm = *reinterpret_cast<AdapterSmem<kTiles>*>(raw);
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int cta = static_cast<int>(blockIdx.x), which = static_cast<int>(blockIdx.y), clusters = static_cast<int>(gridDim.y);
    const __nv_bfloat16* base = static_cast<const __nv_bfloat16*>(p.base);
    __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.out);
    const int rank = p.rank;
    int* ids = sm.ids;
    if (tid < kAdapterRows) sm.rows[tid] = -1;
    if (tid == 0) sm.lead = -1;
    pdl_wait();
    pdl_launch_dependents();
    int id = -1;
    if (tid < p.m) {
        id = p.ids[tid];
        if (id >= p.count) {
            if (cta == 0 && which == 0) report_index(p.status, tid, kIndexAdapter, id);
            id = -1;
        }
    }
    ids[tid] = id;
    // Rows of the same adapter in front of this thread's row: in its warp, and, from each warp's list of adapters and how many
    // rows each has, in the warps in front; eight entries of every list at once. (256 rows of 8 adapters: comparing single rows
    // took 2 us, one list after the other 1.1.)
    const uint32_t fellows = __match_any_sync(0xFFFFFFFFu, id), in_front = (1u << lane) - 1;
    int before = __popc(fellows & in_front);
    const uint32_t firsts = __ballot_sync(0xFFFFFFFFu, before == 0 && id >= 0);
    const int kinds = __popc(firsts);
    if (before == 0 && id >= 0) sm.kinds[warp][__popc(firsts & in_front)] = make_int2(id, __popc(fellows));
    if (lane >= kinds) sm.kinds[warp][lane] = make_int2(-1, 0);
    if (lane == 0) sm.kind_count[warp] = kinds;
    const bool some_without = __syncthreads_or(tid < p.m && id < 0);
    if (warp > 0 && warp * 32 < p.m) {
        constexpr int kAtOnce = 8;
        int most = 0;
#pragma unroll
        for (int w = 0; w < kWarps - 1; ++w) most = max(most, w < warp ? sm.kind_count[w] : 0);
        for (int i = 0; i < most; i += kAtOnce) {
#pragma unroll
            for (int w = 0; w < kWarps - 1; ++w) {
                if (w >= warp) break;
#pragma unroll
                for (int j = 0; j < kAtOnce; ++j) {
                    const int2 kind = sm.kinds[w][i + j];
                    before += kind.x == id ? kind.y : 0;
                }
            }
        }
    }
    const bool leads = id >= 0 && before % kAdapterRows == 0;
    const uint32_t leaders = __ballot_sync(0xFFFFFFFFu, leads);
    if (lane == 0) sm.leads[warp] = leaders;
    // Rows without an adapter: out = base, shared out among the clusters.
    if (base != out && some_without) {
        for (int row = which; row < p.m; row += clusters) {
            if (ids[row] >= 0) continue;
            for (int c = cta * kThreads + tid; c < p.n / 8; c += kAdapterCtas * kThreads)
                *reinterpret_cast<uint4*>(out + row * p.ldo + c * 8) = *reinterpret_cast<const uint4*>(base + row * p.ldb + c * 8);
        }
    }
    __syncthreads();
    if (leads) {
        int place = __popc(leaders & ((1u << lane) - 1));  // leaders in front of this row
        for (int w = 0; w < warp; ++w) place += __popc(sm.leads[w]);
        if (place == which) sm.lead = tid, sm.lead_before = before;
    }
    __syncthreads();
    const int lead = sm.lead;
    if (lead < 0) return;  // fewer leaders than clusters; uniform over the cluster
    const int adapter = ids[lead], at = before - sm.lead_before;
    if (id == adapter && at >= 0 && at < kAdapterRows) sm.rows[at] = tid;
    __syncthreads();
    const int row0 = sm.rows[g], row1 = sm.rows[g + 8];

    // -- x A^T over this CTA's part of k: units of 32, a lane's 16 bytes are two k16 steps' operands -----------------
    {
        const __nv_bfloat16* x0 = static_cast<const __nv_bfloat16*>(p.x) + (row0 < 0 ? 0 : row0) * p.ldx;
        const __nv_bfloat16* x1 = static_cast<const __nv_bfloat16*>(p.x) + (row1 < 0 ? 0 : row1) * p.ldx;
        const __nv_bfloat16* a = static_cast<const __nv_bfloat16*>(p.a) + static_cast<size_t>(adapter) * rank * p.k;
        const int units = (p.k + 31) / 32;
        const int u0 = units * cta / kAdapterCtas, u1 = units * (cta + 1) / kAdapterCtas;
        float acc[kTiles][4] = {};
        const uint4 zero = make_uint4(0, 0, 0, 0);
#pragma unroll(kTiles <= 4 ? 4 : 2)
        for (int u = u0 + warp; u < u1; u += kWarps) {
            const int at = u * 32 + t * 8;
            const bool in = at < p.k;
            const uint4 r0 = in && row0 >= 0 ? *reinterpret_cast<const uint4*>(x0 + at) : zero;
            const uint4 r1 = in && row1 >= 0 ? *reinterpret_cast<const uint4*>(x1 + at) : zero;
            uint4 w[kTiles];
#pragma unroll
            for (int i = 0; i < kTiles; ++i)
                w[i] = in && i * 8 + g < rank ? *reinterpret_cast<const uint4*>(a + static_cast<size_t>(i * 8 + g) * p.k + at) : zero;
            const uint32_t lo[4] = {r0.x, r1.x, r0.y, r1.y}, hi[4] = {r0.z, r1.z, r0.w, r1.w};
#pragma unroll
            for (int i = 0; i < kTiles; ++i) {
                mma_16816<__nv_bfloat16>(acc[i], lo, w[i].x, w[i].y);
                mma_16816<__nv_bfloat16>(acc[i], hi, w[i].z, w[i].w);
            }
        }
#pragma unroll
        for (int i = 0; i < kTiles; ++i) {
            *reinterpret_cast<float2*>(&sm.part[warp][g][i * 8 + 2 * t]) = make_float2(acc[i][0], acc[i][1]);
            *reinterpret_cast<float2*>(&sm.part[warp][g + 8][i * 8 + 2 * t]) = make_float2(acc[i][2], acc[i][3]);
        }
    }
    // -- the second product's operands: groups of 32 columns. Tile j's column c stands for column 8 (c / 2) + 2 j + c % 2 of
    // the group, so that a lane's results of four tiles are eight neighbouring columns: 16 bytes of the output row.
    constexpr int kSteps = (kTiles + 1) / 2;  // k16 steps; a lane's 8 bytes of B are one step's operand
    const __nv_bfloat16* b = static_cast<const __nv_bfloat16*>(p.b) + static_cast<size_t>(adapter) * p.n * rank;
    const int groups = (p.n + 31) / 32;
    uint2 w[kSteps][4];
    uint4 old[2];
    auto fetch = [&](int group) {
        const int column0 = group * 32 + 8 * (g / 2) + (g & 1);  // of tile 0
        const bool col_in = group * 32 + 8 * (g / 2) < p.n;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const bool in = col_in && s * 16 + t * 4 < rank;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                w[s][j] = in ? *reinterpret_cast<const uint2*>(b + static_cast<size_t>(column0 + 2 * j) * rank + s * 16 + t * 4) : make_uint2(0, 0);
        }
        const int column = group * 32 + 8 * t;
        const uint4 zero = make_uint4(0, 0, 0, 0);
        old[0] = column < p.n && row0 >= 0 ? *reinterpret_cast<const uint4*>(base + row0 * p.ldb + column) : zero;
        old[1] = column < p.n && row1 >= 0 ? *reinterpret_cast<const uint4*>(base + row1 * p.ldb + column) : zero;
    };
    int group = cta + warp * kAdapterCtas;  // neighbouring groups in different CTAs: all have work where groups are few
    if (group < groups) fetch(group);
    __syncthreads();
    for (int i = tid; i < kAdapterRows * kTiles * 8; i += kThreads) {
        const int r = i / (kTiles * 8), c = i - r * (kTiles * 8);
        float v = 0.f;
#pragma unroll
        for (int from = 0; from < kWarps; ++from) v += sm.part[from][r][c];
        sm.sum[r][c] = v;
    }
    cluster.sync();
    // -- the cluster's sum, scaled, as BF16 pairs of high and low part (16 bits of mantissa between them) ------------
    {
        const float scale = p.scales[adapter];
        for (int i = tid; i < kAdapterRows * kTiles * 4; i += kThreads) {
            const int r = i / (kTiles * 4), c = (i - r * (kTiles * 4)) * 2;
            float2 s[kAdapterCtas], v = make_float2(0.f, 0.f);
#pragma unroll
            for (int from = 0; from < kAdapterCtas; ++from)
                s[from] = *reinterpret_cast<const float2*>(cluster.map_shared_rank(&sm.sum[r][c], from));
#pragma unroll
            for (int from = 0; from < kAdapterCtas; ++from) v.x += s[from].x, v.y += s[from].y;
            v.x *= scale, v.y *= scale;
            const float2 h = make_float2(high_part(v.x), high_part(v.y));
            sm.high[r][c / 2] = narrow2<__nv_bfloat16>(h.x, h.y);
            sm.low[r][c / 2] = narrow2<__nv_bfloat16>(low_part(v.x, h.x), low_part(v.y, h.y));
        }
    }
    auto read_all = cluster.barrier_arrive();  // no CTA leaves while another still reads its sums
    __syncthreads();
    uint32_t high[kSteps][4], low[kSteps][4];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
        const int at = s * 8 + t * 2;  // pair index: elements 16 s + 4 t .. + 3
        const bool in = at * 2 < rank;
        high[s][0] = in ? sm.high[g][at] : 0, high[s][1] = in ? sm.high[g + 8][at] : 0;
        high[s][2] = in ? sm.high[g][at + 1] : 0, high[s][3] = in ? sm.high[g + 8][at + 1] : 0;
        low[s][0] = in ? sm.low[g][at] : 0, low[s][1] = in ? sm.low[g + 8][at] : 0;
        low[s][2] = in ? sm.low[g][at + 1] : 0, low[s][3] = in ? sm.low[g + 8][at + 1] : 0;
    }
    while (group < groups) {
        float acc[4][4] = {};
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                mma_16816<__nv_bfloat16>(acc[j], high[s], w[s][j].x, w[s][j].y);
                mma_16816<__nv_bfloat16>(acc[j], low[s], w[s][j].x, w[s][j].y);
            }
        }
        const int column = group * 32 + 8 * t;
        const uint4 before_add[2] = {old[0], old[1]};
        group += kAdapterCtas * kWarps;
        if (group < groups) fetch(group);
        if (column < p.n) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int row = half ? row1 : row0;
                if (row < 0) continue;
                float v[kVec] = {};
                add_bf16x8(v, before_add[half]);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[2 * j] += acc[j][2 * half], v[2 * j + 1] += acc[j][2 * half + 1];
                *reinterpret_cast<uint4*>(out + row * p.ldo + column) = pack_bf16x8(v);
            }
        }
    }
    cluster.barrier_wait(std::move(read_all));
}

int launch_adapters(const DlmAdapters& p, const LaunchOpts& o) {
    void* args[] = {const_cast<DlmAdapters*>(&p)};
    auto run = [&](auto tiles) {
        constexpr int kTiles = decltype(tiles)::value;
        const int leaders = p.count + p.m / kAdapterRows;
        return launch_kernel<adapters_kernel<kTiles>>(dim3(kAdapterCtas, leaders < p.m ? leaders : p.m),
                                                      dim3(kThreads),
                                                      static_cast<int>(sizeof(AdapterSmem<kTiles>)), args, o, kAdapterCtas);
    };
    const int tiles = p.rank / 8;
    if (tiles <= 1) return run(std::integral_constant<int, 1>{});
    if (tiles <= 2) return run(std::integral_constant<int, 2>{});
    if (tiles <= 4) return run(std::integral_constant<int, 4>{});
    if (tiles <= 8) return run(std::integral_constant<int, 8>{});
    return run(std::integral_constant<int, 16>{});
}

}  // namespace dlm
