// Low-rank adapters of many requests beside a shared projection:
//
//   out[i] = base[i] + scale[id] * (x[i] A[id]^T) B[id]^T,   id = ids[i]
//
// Bound by reading the adapters' matrices once (rank * (k + n) * 2 bytes each) and, for the small sizes of a block of
// rows, by the chain of latencies between the two products. One launch does both: a cluster of eight CTAs takes up to 16
// rows of one adapter (the M of an mma.sync). Its CTAs split k for x A^T, add their FP32 partial sums through each other's
// shared memory in rank order (so the value never depends on timing), and split n for the second product.
//
// Which rows form a cluster is read off `ids` by the cluster itself: cluster c leads if row c is the 1st, 17th, 33rd ...
// row of its adapter, and then takes the next rows of that adapter, up to 16; otherwise it has nothing to do. No sort, no
// host round trip, any order of ids.
#include <cooperative_groups.h>

#include "mma.cuh"
#include "serving.cuh"

namespace dlm {

namespace {

constexpr int kAdapterThreads = 256;
constexpr int kAdapterWarps = kAdapterThreads / 32;
constexpr int kAdapterCtas = 8;
constexpr int kAdapterRows = 16;
constexpr int kMaxRank = 128;

struct AdapterSmem {
    float part[kAdapterWarps][kAdapterRows][kMaxRank];
    float sum[kAdapterRows][kMaxRank];                     // this CTA's share of x A^T, read by the cluster
    uint32_t high[kAdapterRows][kMaxRank / 2 + 4];         // x A^T times the scale, BF16 pairs
    uint32_t low[kAdapterRows][kMaxRank / 2 + 4];          // what those leave over, BF16 pairs
    int rows[kAdapterRows];
    uint32_t match[kAdapterWarps];
};

}  // namespace

// kTiles: n8 tiles of the first product's output, rank / 8 rounded up.
template <int kTiles>
__global__ void __launch_bounds__(kAdapterThreads) adapters_kernel(const __grid_constant__ DlmAdapters p) {
    namespace cg = cooperative_groups;
    extern __shared__ __align__(16) uint8_t raw[];
    AdapterSmem& sm = *reinterpret_cast<AdapterSmem*>(raw);
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int cta = static_cast<int>(blockIdx.x), lead = static_cast<int>(blockIdx.y);
    pdl_wait();
    pdl_launch_dependents();
    const int lead_id = p.ids[lead];
    const __nv_bfloat16* base = static_cast<const __nv_bfloat16*>(p.base);
    __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.out);
    if (lead_id < 0 || lead_id >= p.count) {  // uniform over the cluster
        if (lead_id >= p.count && cta == 0 && tid == 0) report_index(p.status, lead, kIndexAdapter, lead_id);
        if (base != out) {
            for (int c = cta * kAdapterThreads + tid; c < p.n / 8; c += kAdapterCtas * kAdapterThreads)
                *reinterpret_cast<uint4*>(out + lead * p.ldo + c * 8) = *reinterpret_cast<const uint4*>(base + lead * p.ldb + c * 8);
        }
        return;
    }
    // Rows of this adapter: how many are in front of `lead`, and the 16 from it on.
    {
        const bool same = tid < p.m && p.ids[tid] == lead_id;
        const uint32_t bits = __ballot_sync(0xFFFFFFFFu, same);
        if (lane == 0) sm.match[warp] = bits;
        if (tid < kAdapterRows) sm.rows[tid] = -1;
        __syncthreads();
        int before_me = __popc(bits & ((1u << lane) - 1)), before_lead = 0;
#pragma unroll
        for (int w = 0; w < kAdapterWarps; ++w) {
            if (w < warp) before_me += __popc(sm.match[w]);
            if (w < lead / 32) before_lead += __popc(sm.match[w]);
            if (w == lead / 32) before_lead += __popc(sm.match[w] & ((1u << (lead & 31)) - 1));
        }
        if (before_lead % kAdapterRows) return;  // another cluster has this row; uniform over the cluster
        const int at = before_me - before_lead;
        if (same && at >= 0 && at < kAdapterRows) sm.rows[at] = tid;
        __syncthreads();
    }
    const int row0 = sm.rows[g], row1 = sm.rows[g + 8];
    const int rank = p.rank;

    // -- x A^T over this CTA's part of k: units of 32, a lane's 16 bytes are two k16 steps' operands -----------------
    {
        const __nv_bfloat16* x0 = static_cast<const __nv_bfloat16*>(p.x) + (row0 < 0 ? 0 : row0) * p.ldx;
        const __nv_bfloat16* x1 = static_cast<const __nv_bfloat16*>(p.x) + (row1 < 0 ? 0 : row1) * p.ldx;
        const __nv_bfloat16* a = static_cast<const __nv_bfloat16*>(p.a) + static_cast<size_t>(lead_id) * rank * p.k;
        const int units = (p.k + 31) / 32;
        const int u0 = units * cta / kAdapterCtas, u1 = units * (cta + 1) / kAdapterCtas;
        float acc[kTiles][4] = {};
        const uint4 zero = make_uint4(0, 0, 0, 0);
#pragma unroll 2
        for (int u = u0 + warp; u < u1; u += kAdapterWarps) {
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
    __syncthreads();
    for (int i = tid; i < kAdapterRows * kTiles * 8; i += kAdapterThreads) {
        const int r = i / (kTiles * 8), c = i - r * (kTiles * 8);
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < kAdapterWarps; ++w) v += sm.part[w][r][c];
        sm.sum[r][c] = v;
    }
    cluster.sync();
    // -- the cluster's sum, scaled, as BF16 pairs of high and low part (16 bits of mantissa between them) ------------
    {
        const float scale = p.scales[lead_id];
        for (int i = tid; i < kAdapterRows * kTiles * 4; i += kAdapterThreads) {
            const int r = i / (kTiles * 4), c = (i - r * (kTiles * 4)) * 2;
            float2 v = make_float2(0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kAdapterCtas; ++w) {
                const float2 s = *reinterpret_cast<const float2*>(cluster.map_shared_rank(&sm.sum[r][c], w));
                v.x += s.x, v.y += s.y;
            }
            v.x *= scale, v.y *= scale;
            const uint32_t high = narrow2<__nv_bfloat16>(v.x, v.y);
            const float2 h = widen2<__nv_bfloat16>(high);
            sm.high[r][c / 2] = high;
            sm.low[r][c / 2] = narrow2<__nv_bfloat16>(v.x - h.x, v.y - h.y);
        }
    }
    cluster.sync();  // also: no CTA leaves while another still reads its sums

    // -- the second product over this CTA's part of n ----------------------------------------------------------------
    // Groups of 32 columns. Tile j's column c stands for column 8 (c / 2) + 2 j + c % 2 of the group, so that a lane's
    // results of four tiles are eight neighbouring columns: 16 bytes of the output row.
    constexpr int kSteps = (kTiles + 1) / 2;  // k16 steps; a lane's 8 bytes of B are one step's operand
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
    const __nv_bfloat16* b = static_cast<const __nv_bfloat16*>(p.b) + static_cast<size_t>(lead_id) * p.n * rank;
    const int groups = (p.n + 31) / 32;
    for (int group = cta * kAdapterWarps + warp; group < groups; group += kAdapterCtas * kAdapterWarps) {
        float acc[4][4] = {};
        const int column0 = group * 32 + 8 * (g / 2) + (g & 1);  // of tile 0
        const bool col_in = group * 32 + 8 * (g / 2) < p.n;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const bool in = col_in && s * 16 + t * 4 < rank;
            uint2 w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                w[j] = in ? *reinterpret_cast<const uint2*>(b + static_cast<size_t>(column0 + 2 * j) * rank + s * 16 + t * 4) : make_uint2(0, 0);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                mma_16816<__nv_bfloat16>(acc[j], high[s], w[j].x, w[j].y);
                mma_16816<__nv_bfloat16>(acc[j], low[s], w[j].x, w[j].y);
            }
        }
        const int column = group * 32 + 8 * t;
        if (column < p.n) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int row = half ? row1 : row0;
                if (row < 0) continue;
                const uint4 old = *reinterpret_cast<const uint4*>(base + row * p.ldb + column);
                float v[kVec] = {};
                add_bf16x8(v, old);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[2 * j] += acc[j][2 * half], v[2 * j + 1] += acc[j][2 * half + 1];
                *reinterpret_cast<uint4*>(out + row * p.ldo + column) = pack_bf16x8(v);
            }
        }
    }
}

int launch_adapters(const DlmAdapters& p, const LaunchOpts& o) {
    void* args[] = {const_cast<DlmAdapters*>(&p)};
    auto run = [&](auto tiles) {
        return launch_kernel<adapters_kernel<decltype(tiles)::value>>(dim3(kAdapterCtas, p.m), dim3(kAdapterThreads),
                                                                      static_cast<int>(sizeof(AdapterSmem)), args, o, kAdapterCtas);
    };
    const int tiles = p.rank / 8;
    if (tiles <= 1) return run(std::integral_constant<int, 1>{});
    if (tiles <= 2) return run(std::integral_constant<int, 2>{});
    if (tiles <= 4) return run(std::integral_constant<int, 4>{});
    if (tiles <= 8) return run(std::integral_constant<int, 8>{});
    return run(std::integral_constant<int, 16>{});
}

}  // namespace dlm
