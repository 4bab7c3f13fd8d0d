// Attention of new tokens over a paged cache of keys and values (dlmrt/ops/triton/attention.py; split over the keys and
// joined as dlmrt/models/sdar/engine.py:127-132 does).
//
//   o = sum_j exp(s_j) v_j / sum_j exp(s_j),   s_j = scale * q . k_j over the keys that the row's token sees
//
// One pass over the keys with a running maximum m and sum l per row: a tile's new maximum m' rescales what is there by
// exp2(m - m') (all exponents in base 2, scale * log2(e) folded into the scores).
//
// The rows that share a key head are its query heads times the new tokens; 16 of them make the M of an mma.sync. A single
// token fills a few rows and is bound by reading the cache, so the tensor instructions only have to keep up with HBM. The
// keys of one sequence are cut into chunks, one CTA each; in a CTA each of four warps takes every fourth tile of 16 keys
// through a ring of its own (cp.async, no block-wide step in the main loop), with its own maximum, sum and output in
// registers. The four are joined in shared memory at the end, and chunks of one sequence by join_kernel.
#include "mma.cuh"
#include "serving.cuh"

namespace dlm {

namespace {

constexpr int kAttendWarps = 4;
constexpr int kTileKeys = 16;
constexpr float kLog2e = 1.4426950408889634f;

// What a row tile of one sequence has to look at: keys [lo, hi), and the same for single tokens.
struct Span {
    int length, first_pos;  // keys of the sequence; position of its first new token
    int lo, hi;             // keys that some row of the tile sees
    int chunks;             // CTAs that have keys, at least 1
    int base;               // first key of chunk 0
};

__device__ __forceinline__ int seen_from(const AttendDev& p, const Span& s, int token) {
    return p.a.window > 0 ? max(0, s.first_pos + token - p.a.window + 1) : 0;
}
__device__ __forceinline__ int seen_to(const AttendDev& p, const Span& s, int token) {
    return p.a.causal ? min(s.length, s.first_pos + token + 1) : s.length;
}

__device__ __forceinline__ Span span_of(const AttendDev& p, int sequence, int row_tile, bool tell) {
    Span s;
    const long long room = static_cast<long long>(p.a.table_pages) << p.page_shift;
    const int length = p.a.lengths[sequence];
    s.length = length < 0 ? 0 : length > room ? static_cast<int>(room) : length;
    if (tell && s.length != length) report_index(p.a.cache.status, sequence, kIndexLength, length);
    s.first_pos = s.length - p.a.tokens;
    const int first = row_tile * kRowTile, last = min(first + kRowTile, p.rows) - 1;
    s.lo = seen_from(p, s, first / p.group);
    s.hi = seen_to(p, s, last / p.group);
    s.base = s.lo & ~(kTileKeys - 1);
    s.chunks = s.hi > s.base ? (s.hi - s.base + p.chunk - 1) / p.chunk : 1;
    return s;
}

// One warp's stage: 16 keys, then 16 values, rows of head_dim elements in 16-byte pieces whose order is permuted by row so
// that ldmatrix (and, for FP8 keys, 16-byte loads of four lanes per row) meets each bank once.
template <int D, bool kCodes>
struct Stage {
    static constexpr int kPieces = D * (kCodes ? 1 : 2) / 16;  // of a row
    static constexpr int kBytes = kTileKeys * kPieces * 16;     // of the keys, or of the values
    __device__ static __forceinline__ int value_piece(int row, int c) {
        return kPieces == 4 ? c ^ ((row >> 1) & 3) : c ^ (row & 7);
    }
    __device__ static __forceinline__ int key_piece(int row, int c) {
        return !kCodes || kPieces == 4 ? value_piece(row, c) : c ^ ((row & 1) << 2);
    }
};

// All-ones in the 16-bit values (FP8: bytes) of a word that are infinite or NaN. E4M3 has no infinity, and one NaN.
template <typename M, bool kCodes>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
    if constexpr (kCodes) return __vcmpeq4(w & 0x7F7F7F7Fu, 0x7F7F7F7Fu);
    constexpr uint32_t kExponent = std::is_same<M, __half>::value ? 0x7C007C00u : 0x7F807F80u;
    return __vcmpeq2(w & kExponent, kExponent);
}

template <int D, bool kCodes>
constexpr int stages() {
    return 3;
}

template <int D, bool kCodes>
constexpr int attend_smem() {
    const int ring = stages<D, kCodes>() * kAttendWarps * 2 * Stage<D, kCodes>::kBytes;
    const int join = kAttendWarps * kRowTile * (D + 4) * 4;
    return ring > join ? ring : join;
}

}  // namespace

// T: type of queries and output. Products are of T, or of halves where the cache holds FP8 codes (every code is a half).
template <typename T, int D, bool kCodes>
__global__ void __launch_bounds__(kAttendWarps * 32) attend_kernel(const __grid_constant__ AttendDev p) {
    using M = typename std::conditional<kCodes, __half, T>::type;
    using S = Stage<D, kCodes>;
    constexpr int kStages = stages<D, kCodes>();
    constexpr int kSteps = D / 16;       // k16 steps of q . k
    constexpr int kOut = D / 8;          // n8 tiles of the output
    constexpr int kElem = kCodes ? 1 : 2;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float warp_stats[kAttendWarps][kRowTile][2];
    __shared__ uint32_t present_keys[kAttendWarps][4];
    __shared__ float weights_of_tile[kAttendWarps][kRowTile][kTileKeys + 1];

    const int warp = uniform(static_cast<int>(threadIdx.x >> 5)), lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const int sequence = blockIdx.z;
    const int head = static_cast<int>(blockIdx.y) / p.row_tiles, row_tile = static_cast<int>(blockIdx.y) - head * p.row_tiles;
    pdl_wait();
    pdl_launch_dependents();
    const Span span = span_of(p, sequence, row_tile, blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0);
    const int chunk = blockIdx.x;
    if (chunk >= span.chunks) return;
    const int start = span.base + chunk * p.chunk;
    const int end = min(span.hi, start + p.chunk);
    const int tiles = end > start ? (end - start + kTileKeys - 1) / kTileKeys : 0;

    // This thread's two rows: g and g + 8 of the tile.
    const int row0 = row_tile * kRowTile + g, row1 = row0 + 8;
    const int token0 = min(row0, p.rows - 1) / p.group, token1 = min(row1, p.rows - 1) / p.group;
    const int from0 = seen_from(p, span, token0), to0 = seen_to(p, span, token0);
    const int from1 = seen_from(p, span, token1), to1 = seen_to(p, span, token1);
    const int last_token = min(row_tile * kRowTile + kRowTile, p.rows) - 1;
    const int all_from = seen_from(p, span, last_token / p.group);               // from here on every row sees the keys
    const int all_to = seen_to(p, span, (row_tile * kRowTile) / p.group);        // up to here

    auto q_row = [&](int row) -> const T* {
        const int token = row / p.group, of = row - token * p.group;
        return static_cast<const T*>(p.a.q) + sequence * p.a.q_strides[0] + token * p.a.q_strides[1] +
               static_cast<long long>(head * p.group + of) * p.a.q_strides[2];
    };
    // Queries as the A operand. With FP8 keys the contraction runs in the order in which a lane's 16-byte piece of a key
    // row holds them: step 4s + j of lane t covers elements 64 s + 16 t + 4 j .. + 3.
    uint32_t q[kSteps][4];
    const bool has0 = row0 < p.rows, has1 = row1 < p.rows;
    const T* q0 = has0 ? q_row(row0) : nullptr;
    const T* q1 = has1 ? q_row(row1) : nullptr;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
        const int at0 = kCodes ? (s / 4) * 64 + t * 16 + (s % 4) * 4 : s * 16 + t * 2;
        const int at1 = at0 + (kCodes ? 2 : 8);
        q[s][0] = has0 ? *reinterpret_cast<const uint32_t*>(q0 + at0) : 0;
        q[s][1] = has1 ? *reinterpret_cast<const uint32_t*>(q1 + at0) : 0;
        q[s][2] = has0 ? *reinterpret_cast<const uint32_t*>(q0 + at1) : 0;
        q[s][3] = has1 ? *reinterpret_cast<const uint32_t*>(q1 + at1) : 0;
    }
    float scale0 = p.a.scale * kLog2e, scale1 = scale0;
    if constexpr (kCodes) {
        // A BF16 row may not fit a half: it is scaled by the power of two that brings its largest element below 2 (exact,
        // but for elements 2^-14 of the largest, whose error is at most 2^-25 of it), and the scores are scaled back.
        const float key_scale = p.a.cache.k_scale[head];
        scale0 *= key_scale, scale1 *= key_scale;
        float top0 = 0.f, top1 = 0.f;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                const float2 a = widen2<T>(q[s][i]), b = widen2<T>(q[s][i + 1]);
                top0 = fmaxf(top0, fmaxf(fabsf(a.x), fabsf(a.y)));
                top1 = fmaxf(top1, fmaxf(fabsf(b.x), fabsf(b.y)));
            }
        }
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
            top0 = fmaxf(top0, __shfl_xor_sync(0xFFFFFFFFu, top0, o));
            top1 = fmaxf(top1, __shfl_xor_sync(0xFFFFFFFFu, top1, o));
        }
        // 2^-e and 2^e for the exponent e of the largest element, kept where both are normal numbers.
        const int e0 = min(max(static_cast<int>(__float_as_uint(top0) >> 23) - 127, -100), 126);
        const int e1 = min(max(static_cast<int>(__float_as_uint(top1) >> 23) - 127, -100), 126);
        const float down0 = __uint_as_float(static_cast<uint32_t>(127 - e0) << 23);
        const float down1 = __uint_as_float(static_cast<uint32_t>(127 - e1) << 23);
        scale0 *= __uint_as_float(static_cast<uint32_t>(127 + e0) << 23);
        scale1 *= __uint_as_float(static_cast<uint32_t>(127 + e1) << 23);
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 a = widen2<T>(q[s][i]);
                const float down = i & 1 ? down1 : down0;
                q[s][i] = narrow2<__half>(a.x * down, a.y * down);
            }
        }
    }

    // -- the ring ---------------------------------------------------------------------------------------------------
    uint8_t* ring = smem + warp * (kStages * 2 * S::kBytes);
    const uint32_t ring_u32 = smem_u32(ring);
    const int32_t* table = p.a.page_table + sequence * p.a.table_stride;
    const uint8_t* keys = static_cast<const uint8_t*>(p.a.cache.keys) + head * p.a.cache.k_strides[1] * kElem;
    const uint8_t* values = static_cast<const uint8_t*>(p.a.cache.values) + head * p.a.cache.v_strides[1] * kElem;
    const long long k_page = p.a.cache.k_strides[0] * kElem, k_slot = p.a.cache.k_strides[2] * kElem;
    const long long v_page = p.a.cache.v_strides[0] * kElem, v_slot = p.a.cache.v_strides[2] * kElem;
    const int slot_mask = (1 << p.page_shift) - 1;

    auto page_of = [&](int it) -> int {  // lane r of the lower half: page of key r of tile `it`, -1 where there is none
        const int key = start + (warp + it * kAttendWarps) * kTileKeys + lane;
        if (lane >= kTileKeys || key >= end) return -1;
        const int page = table[key >> p.page_shift];
        if (page >= 0 && page < p.a.cache.pages) return page;
        if (key >= span.lo) report_index(p.a.cache.status, sequence, kIndexPage, page);
        return -1;
    };
    const int mine = tiles > warp ? (tiles - warp + kAttendWarps - 1) / kAttendWarps : 0;  // tiles of this warp
    int page_ahead = page_of(0);
    auto issue = [&](int it, int stage) {
        if (it < mine) {
            const int page = page_ahead;
            const uint32_t present = __ballot_sync(0xFFFFFFFFu, page >= 0);
            if (lane == 0) present_keys[warp][stage] = present;
            const int key0 = start + (warp + it * kAttendWarps) * kTileKeys;
            const uint32_t to = ring_u32 + stage * 2 * S::kBytes;
            constexpr int kRowsAtOnce = 32 / S::kPieces;
            const int c = lane % S::kPieces, r0 = lane / S::kPieces;
#pragma unroll
            for (int i = 0; i < kTileKeys / kRowsAtOnce; ++i) {
                const int r = r0 + i * kRowsAtOnce;
                const int id = __shfl_sync(0xFFFFFFFFu, page, r);
                const bool there = id >= 0;
                const long long at = there ? id : 0;
                const int slot = (key0 + r) & slot_mask;
                cp_async_16(to + (r * S::kPieces + S::key_piece(r, c)) * 16, keys + at * k_page + slot * k_slot + c * 16, there);
                cp_async_16(to + S::kBytes + (r * S::kPieces + S::value_piece(r, c)) * 16,
                            values + at * v_page + slot * v_slot + c * 16, there);
            }
            page_ahead = page_of(it + 1);
        }
        cp_async_commit();
    };

    float o[kOut][4];
#pragma unroll
    for (int i = 0; i < kOut; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;

#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) issue(s, s);
    int stage = 0, fill = kStages - 1;
    for (int it = 0; it < mine; ++it) {
        cp_async_wait<kStages - 2>();
        __syncwarp();  // every lane's copies of this stage have landed, and every lane is done with the stage before
        issue(it + kStages - 1, fill);
        const int key0 = start + (warp + it * kAttendWarps) * kTileKeys;
        const uint8_t* stage_k = ring + stage * 2 * S::kBytes;
        const uint32_t stage_k32 = ring_u32 + stage * 2 * S::kBytes, stage_v32 = stage_k32 + S::kBytes;
        const uint32_t present = present_keys[warp][stage];

        // scores: columns are keys, 0..7 in s[0], 8..15 in s[1]
        float s[2][4] = {};
        if constexpr (!kCodes) {
            const int r = (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                uint32_t b[4];
                ldmatrix_x4(b, stage_k32 + (r * S::kPieces + S::key_piece(r, 2 * k + ((lane >> 3) & 1))) * 16);
                mma_16816<M>(s[0], q[k], b[0], b[1]);
                mma_16816<M>(s[1], q[k], b[2], b[3]);
            }
        } else {
#pragma unroll
            for (int k4 = 0; k4 < kSteps / 4; ++k4) {
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const int r = g + 8 * n;
                    const uint4 w = *reinterpret_cast<const uint4*>(stage_k + (r * S::kPieces + S::key_piece(r, 4 * k4 + t)) * 16);
                    const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        mma_16816<M>(s[n], q[4 * k4 + j], e4m3x2_to_f16x2(words[j] & 0xFFFFu), e4m3x2_to_f16x2(words[j] >> 16));
                }
            }
        }
        const bool by_row = key0 < all_from || key0 + kTileKeys > all_to;  // rows see different keys of this tile
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            s[n][0] *= scale0, s[n][1] *= scale0, s[n][2] *= scale1, s[n][3] *= scale1;
        }
        if (by_row || present != 0xFFFFu) {
#pragma unroll
            for (int n = 0; n < 2; ++n) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int c = 8 * n + 2 * t + e, key = key0 + c;
                    const bool there = (present >> c) & 1;
                    if (!there || key < from0 || key >= to0) s[n][e] = -INFINITY;
                    if (!there || key < from1 || key >= to1) s[n][2 + e] = -INFINITY;
                }
            }
        }
        float top0 = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1]));
        float top1 = fmaxf(fmaxf(s[0][2], s[0][3]), fmaxf(s[1][2], s[1][3]));
#pragma unroll
        for (int x = 1; x < 4; x <<= 1) {
            top0 = fmaxf(top0, __shfl_xor_sync(0xFFFFFFFFu, top0, x));
            top1 = fmaxf(top1, __shfl_xor_sync(0xFFFFFFFFu, top1, x));
        }
        if (__any_sync(0xFFFFFFFFu, top0 > m0 || top1 > m1)) {
            const float n0 = fmaxf(m0, top0), n1 = fmaxf(m1, top1);
            const float f0 = m0 == n0 ? 1.f : exp2_approx(m0 - n0), f1 = m1 == n1 ? 1.f : exp2_approx(m1 - n1);
            m0 = n0, m1 = n1;
            l0 *= f0, l1 *= f1;
#pragma unroll
            for (int i = 0; i < kOut; ++i) o[i][0] *= f0, o[i][1] *= f0, o[i][2] *= f1, o[i][3] *= f1;
        }
        const float sub0 = m0 == -INFINITY ? 0.f : m0, sub1 = m1 == -INFINITY ? 0.f : m1;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            s[n][0] = exp2_approx(s[n][0] - sub0), s[n][1] = exp2_approx(s[n][1] - sub0);
            s[n][2] = exp2_approx(s[n][2] - sub1), s[n][3] = exp2_approx(s[n][3] - sub1);
            l0 += s[n][0] + s[n][1], l1 += s[n][2] + s[n][3];
        }

        // Values that are not finite, in a key that some rows see and others do not: 0 * inf would reach the others. They
        // are added here to the rows that see them, and are zero in the product below.
        if (by_row) {
            uint32_t* words = reinterpret_cast<uint32_t*>(ring + stage * 2 * S::kBytes + S::kBytes);
            bool apart = false;
            for (int i = lane; i < S::kBytes / 4; i += 32) apart |= not_finite<M, kCodes>(words[i]) != 0;
            if (__any_sync(0xFFFFFFFFu, apart)) {
                float (&w)[kRowTile][kTileKeys + 1] = weights_of_tile[warp];
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    w[g][8 * n + 2 * t] = s[n][0], w[g][8 * n + 2 * t + 1] = s[n][1];
                    w[g + 8][8 * n + 2 * t] = s[n][2], w[g + 8][8 * n + 2 * t + 1] = s[n][3];
                }
                __syncwarp();
#pragma unroll 1
                for (int c = 0; c < kTileKeys; ++c) {
                    const int key = key0 + c;
                    const bool there = (present >> c) & 1;
                    const bool see0 = there && key >= from0 && key < to0, see1 = there && key >= from1 && key < to1;
                    const float w0 = w[g][c], w1 = w[g + 8][c];
#pragma unroll
                    for (int i = 0; i < kOut; ++i) {
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int byte = (kCodes ? (i / 2) * 16 + 4 * t + 2 * e + (i & 1) : 8 * i + 2 * t + e) * kElem;
                            const uint8_t* at = stage_k + S::kBytes + (c * S::kPieces + S::value_piece(c, byte / 16)) * 16 + byte % 16;
                            float v;
                            if constexpr (kCodes) v = widen2<__half>(e4m3x2_to_f16x2(*at)).x;
                            else v = widen2<M>(*reinterpret_cast<const uint16_t*>(at)).x;
                            if (!isfinite(v)) {
                                if (see0) o[i][e] += w0 * v;
                                if (see1) o[i][2 + e] += w1 * v;
                            }
                        }
                    }
                }
                __syncwarp();
                for (int i = lane; i < S::kBytes / 4; i += 32) words[i] &= ~not_finite<M, kCodes>(words[i]);
                __syncwarp();
            }
        }
        {
            uint32_t a[4] = {narrow2<M>(s[0][0], s[0][1]), narrow2<M>(s[0][2], s[0][3]), narrow2<M>(s[1][0], s[1][1]),
                             narrow2<M>(s[1][2], s[1][3])};
            const int r = (lane & 7) + (((lane >> 3) & 1) << 3);
#pragma unroll
            for (int i = 0; i < S::kPieces / 2; ++i) {
                uint32_t b[4];
                ldmatrix_x4_trans(b, stage_v32 + (r * S::kPieces + S::value_piece(r, 2 * i + (lane >> 4))) * 16);
                if constexpr (!kCodes) {
                    mma_16816<M>(o[2 * i], a, b[0], b[1]);
                    mma_16816<M>(o[2 * i + 1], a, b[2], b[3]);
                } else {
                    // b[0], b[1]: keys 2t, 2t + 1 (+ 8) of elements 2g and 2g + 1 of a 16-byte piece; b[2], b[3]: the next
                    // piece. One product takes the even elements, one the odd ones.
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const uint32_t even0 = __byte_perm(b[2 * c], 0, 0x4420), odd0 = __byte_perm(b[2 * c], 0, 0x4431);
                        const uint32_t even1 = __byte_perm(b[2 * c + 1], 0, 0x4420), odd1 = __byte_perm(b[2 * c + 1], 0, 0x4431);
                        mma_16816<M>(o[4 * i + 2 * c], a, e4m3x2_to_f16x2(even0), e4m3x2_to_f16x2(even1));
                        mma_16816<M>(o[4 * i + 2 * c + 1], a, e4m3x2_to_f16x2(odd0), e4m3x2_to_f16x2(odd1));
                    }
                }
            }
        }
        if (++stage == kStages) stage = 0;
        if (++fill == kStages) fill = 0;
    }

    // -- the four warps' results ------------------------------------------------------------------------------------
#pragma unroll
    for (int x = 1; x < 4; x <<= 1) {
        l0 += __shfl_xor_sync(0xFFFFFFFFu, l0, x);
        l1 += __shfl_xor_sync(0xFFFFFFFFu, l1, x);
    }
    if (t == 0) {
        warp_stats[warp][g][0] = m0, warp_stats[warp][g][1] = l0;
        warp_stats[warp][g + 8][0] = m1, warp_stats[warp][g + 8][1] = l1;
    }
    cp_async_wait<0>();
    __syncthreads();  // statistics are there, and nobody reads or fills the ring any more
    constexpr int kPitch = D + 4;
    float* joined = reinterpret_cast<float*>(smem);
    {
        float n0 = -INFINITY, n1 = -INFINITY;
#pragma unroll
        for (int w = 0; w < kAttendWarps; ++w) n0 = fmaxf(n0, warp_stats[w][g][0]), n1 = fmaxf(n1, warp_stats[w][g + 8][0]);
        const float f0 = m0 == -INFINITY ? 0.f : exp2_approx(m0 - n0), f1 = m1 == -INFINITY ? 0.f : exp2_approx(m1 - n1);
        // A warp that met no visible key has all zeros, or NaN times zero from a score that was NaN: kept as it is.
        float* to = joined + warp * kRowTile * kPitch;
#pragma unroll
        for (int i = 0; i < kOut; ++i) {
            if constexpr (!kCodes) {
                *reinterpret_cast<float2*>(to + g * kPitch + 8 * i + 2 * t) = make_float2(o[i][0] * f0, o[i][1] * f0);
                *reinterpret_cast<float2*>(to + (g + 8) * kPitch + 8 * i + 2 * t) = make_float2(o[i][2] * f1, o[i][3] * f1);
            } else {
                const int d = (i / 2) * 16 + 4 * t + (i & 1);
                to[g * kPitch + d] = o[i][0] * f0, to[g * kPitch + d + 2] = o[i][1] * f0;
                to[(g + 8) * kPitch + d] = o[i][2] * f1, to[(g + 8) * kPitch + d + 2] = o[i][3] * f1;
            }
        }
    }
    __syncthreads();
    const int rows = min(kRowTile, p.rows - row_tile * kRowTile);
    const bool whole = span.chunks == 1;
    const size_t piece = ((static_cast<size_t>(sequence) * p.a.cache.heads + head) * p.row_tiles + row_tile) * p.chunks + chunk;
    const float value_scale = kCodes ? p.a.cache.v_scale[head] : 1.f;
    for (int i = threadIdx.x; i < rows * (D / 4); i += kAttendWarps * 32) {
        const int r = i / (D / 4), d = (i - r * (D / 4)) * 4;
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        float top = -INFINITY, l = 0.f;
#pragma unroll
        for (int w = 0; w < kAttendWarps; ++w) {
            const float4 v = *reinterpret_cast<const float4*>(joined + (w * kRowTile + r) * kPitch + d);
            sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
            top = fmaxf(top, warp_stats[w][r][0]);
        }
#pragma unroll
        for (int w = 0; w < kAttendWarps; ++w) {
            const float m = warp_stats[w][r][0];
            l += warp_stats[w][r][1] * (m == -INFINITY ? 0.f : exp2_approx(m - top));
        }
        if (whole) {
            const float inv = l == 0.f ? 0.f : value_scale / l;
            const int row = row_tile * kRowTile + r, token = row / p.group, of = row - token * p.group;
            T* out = static_cast<T*>(p.a.out) + sequence * p.a.out_strides[0] + token * p.a.out_strides[1] +
                     static_cast<long long>(head * p.group + of) * p.a.out_strides[2] + d;
            *reinterpret_cast<uint2*>(out) = make_uint2(narrow2<T>(sum.x * inv, sum.y * inv), narrow2<T>(sum.z * inv, sum.w * inv));
            if (p.a.lse != nullptr && d == 0)
                p.a.lse[(static_cast<size_t>(sequence) * p.a.tokens + token) * p.a.q_heads + head * p.group + of] =
                    l == 0.f ? -INFINITY : (top + log2f(l)) * (1.f / kLog2e);
        } else {
            *reinterpret_cast<float4*>(p.partial + (piece * p.rows_cap + r) * D + d) = sum;
            if (d == 0) *reinterpret_cast<float2*>(p.stats + (piece * p.rows_cap + r) * 2) = make_float2(top, l);
        }
    }
}

// Joins the chunks of one row: out = sum_c exp2(m_c - m) o_c / sum_c exp2(m_c - m) l_c. One block per row; D / 4 threads
// cover a row, the block's other threads further chunks.
constexpr int kJoinThreads = 256;

template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const __grid_constant__ AttendDev p) {
    constexpr int kAcross = D / 4, kDeep = kJoinThreads / kAcross;
    __shared__ float4 sums[kDeep][kAcross];
    __shared__ float ls[kDeep];
    const int r = blockIdx.x, sequence = blockIdx.z;
    const int head = static_cast<int>(blockIdx.y) / p.row_tiles, row_tile = static_cast<int>(blockIdx.y) - head * p.row_tiles;
    const int row = row_tile * kRowTile + r;
    if (row >= p.rows) return;
    pdl_wait();
    pdl_launch_dependents();
    const Span span = span_of(p, sequence, row_tile, false);
    if (span.chunks == 1) return;
    const size_t piece = ((static_cast<size_t>(sequence) * p.a.cache.heads + head) * p.row_tiles + row_tile) * p.chunks;
    const int x = threadIdx.x % kAcross, y = threadIdx.x / kAcross;
    const float* stats = p.stats + (piece * p.rows_cap + r) * 2;
    const float* partial = p.partial + (piece * p.rows_cap + r) * D + x * 4;
    float top = -INFINITY;
    for (int c = 0; c < span.chunks; ++c) top = fmaxf(top, __ldcg(stats + static_cast<size_t>(c) * p.rows_cap * 2));
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
    for (int c = y; c < span.chunks; c += kDeep) {
        const float2 ml = __ldcg(reinterpret_cast<const float2*>(stats + static_cast<size_t>(c) * p.rows_cap * 2));
        const float4 v = __ldcg(reinterpret_cast<const float4*>(partial + static_cast<size_t>(c) * p.rows_cap * D));
        const float f = ml.x == -INFINITY ? 0.f : exp2_approx(ml.x - top);
        l += ml.y * f;
        sum.x += v.x * f, sum.y += v.y * f, sum.z += v.z * f, sum.w += v.w * f;
    }
    sums[y][x] = sum;
    if (x == 0) ls[y] = l;
    __syncthreads();
    if (y != 0) return;
#pragma unroll
    for (int i = 1; i < kDeep; ++i) {
        const float4 v = sums[i][x];
        sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
        l += ls[i];
    }
    const float value_scale = p.a.cache.type == DLM_E4M3 ? p.a.cache.v_scale[head] : 1.f;
    const float inv = l == 0.f ? 0.f : value_scale / l;
    const int token = row / p.group, of = row - token * p.group;
    T* out = static_cast<T*>(p.a.out) + sequence * p.a.out_strides[0] + token * p.a.out_strides[1] +
             static_cast<long long>(head * p.group + of) * p.a.out_strides[2] + x * 4;
    *reinterpret_cast<uint2*>(out) = make_uint2(narrow2<T>(sum.x * inv, sum.y * inv), narrow2<T>(sum.z * inv, sum.w * inv));
    if (p.a.lse != nullptr && x == 0)
        p.a.lse[(static_cast<size_t>(sequence) * p.a.tokens + token) * p.a.q_heads + head * p.group + of] =
            l == 0.f ? -INFINITY : (top + log2f(l)) * (1.f / kLog2e);
}

template <typename T, int D>
static int launch_attend_d(const AttendDev& p, const LaunchOpts& o) {
    void* args[] = {const_cast<AttendDev*>(&p)};
    const dim3 grid(p.chunks, p.a.cache.heads * p.row_tiles, p.a.batch), block(kAttendWarps * 32);
    const int rc = p.a.cache.type == DLM_E4M3 ? launch_kernel<attend_kernel<T, D, true>>(grid, block, attend_smem<D, true>(), args, o)
                                              : launch_kernel<attend_kernel<T, D, false>>(grid, block, attend_smem<D, false>(), args, o);
    if (rc != 0 || p.chunks == 1) return rc;
    return launch_kernel<join_kernel<T, D>>(dim3(p.rows_cap, p.a.cache.heads * p.row_tiles, p.a.batch), dim3(kJoinThreads), 0, args,
                                            {o.stream, true, false});  // always a dependent launch of the kernel above
}

int launch_attend(const AttendDev& p, const LaunchOpts& o) {
    auto by_dim = [&](auto t) {
        using T = decltype(t);
        switch (p.a.cache.head_dim) {
            case 64: return launch_attend_d<T, 64>(p, o);
            case 128: return launch_attend_d<T, 128>(p, o);
            default: return launch_attend_d<T, 256>(p, o);
        }
    };
    return p.a.type == DLM_F16 ? by_dim(__half{}) : by_dim(__nv_bfloat16{});
}

}  // namespace dlm
