// Attention of new tokens over a paged cache of keys and values (dlmrt/ops/triton/attention.py; split over the keys and
// joined as dlmrt/models/sdar/engine.py:127-132 does).
//
//   o = sum_j exp(s_j) v_j / sum_j exp(s_j),   s_j = scale * q . k_j over the keys that the row's token sees
//
// One pass over the keys with a running maximum m and sum l per row: a tile's new maximum m' rescales what is there by
// exp2(m - m') (all exponents in base 2, scale * log2(e) folded into the scores).
//
// The rows that share a key head are its query heads times the new tokens; 16 of them make the M of an mma.sync. A single
// token fills a few rows and is bound by reading the cache, so the tensor instructions only have to keep up with HBM.
//
//   warp 4     deals out the work and requests keys and values: steps of 64 keys into a ring of stages, as TMA boxes of a
//              page's slots (pages in any order; up to 64 slots a box). See paged_attend.cuh.
//   warps 0-3  take 16 keys of every step each, with their own maximum, sum and output in registers: no step in which they
//              wait for one another but an item's end, where the four are joined in shared memory.
//
// Many rows (a block of tokens) are another kernel's (paged_blocks.cu).
#include "paged_attend.cuh"

namespace dlm {

namespace {

constexpr int kConsumers = 4;                            // warps that compute
constexpr int kAttendThreads = (kConsumers + 1) * 32;
constexpr int kWarpKeys = kTileKeys / kConsumers;        // 16

// A stage: 64 keys, then 64 values, as TMA writes them: box by box (a page's slots, at most 64), in a box column blocks of up
// to 128 bytes, in each the rows one after the other with their 16-byte pieces permuted by row (the 128- or 64-byte swizzle),
// so that ldmatrix meets each bank once.
template <int D, bool kCodes>
struct Stage {
    static constexpr int kPieces = D * (kCodes ? 1 : 2) / 16;           // 16-byte pieces of a row
    static constexpr int kBytes = kTileKeys * kPieces * 16;              // of the keys, or of the values
    static constexpr int kAcross = kPieces < 8 ? kPieces : 8;            // pieces of a column block's row
    int first;   // offset of a warp's first row
    int half;    // from its row r to row r + 8: in the same box, or (pages of 8) in the next
    int block;   // from a column block to the next
    __device__ __forceinline__ Stage(int box_keys, int row)
        : first(row / box_keys * box_keys * kPieces * 16 + row % box_keys * kAcross * 16),
          half(box_keys == 8 ? 8 * kPieces * 16 : 8 * kAcross * 16), block(box_keys * kAcross * 16) {}
    // Offset of a piece of the warp's row `row`, 0 to 15.
    __device__ __forceinline__ int at(int row, int piece) const {
        const int turn = kAcross == 8 ? row & 7 : (row >> 1) & 3;
        return first + (piece / kAcross) * block + (row >> 3) * half + (row & 7) * (kAcross * 16) + ((piece % kAcross) ^ turn) * 16;
    }
};

// All-ones in the 16-bit values (FP8: bytes) of a word that are infinite or NaN. E4M3 has no infinity, and one NaN.
template <typename M, bool kCodes>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
    if constexpr (kCodes) return __vcmpeq4(w & 0x7F7F7F7Fu, 0x7F7F7F7Fu);
    constexpr uint32_t kExponent = std::is_same<M, __half>::value ? 0x7C007C00u : 0x7F807F80u;
    return __vcmpeq2(w & kExponent, kExponent);
}

// Shared memory of a CTA, and how many CTAs an SM holds of it (registers are held to what they leave each other).
template <int D, bool kCodes>
struct AttendSmem {
    static constexpr int kCtas = D == 64 ? 3 : D == 256 && !kCodes ? 1 : 2;
    static constexpr int kStages = D == 64 ? (kCodes ? 6 : 4) : D == 128 && kCodes ? 6 : 3;
    static constexpr int kRing = kStages * 2 * Stage<D, kCodes>::kBytes;
    static constexpr int kPitch = D + 4;
    static constexpr int kJoinRows = D == 256 ? 2 : 4;  // rows of a tile that the warps exchange at a time
    static constexpr int kJoin = kConsumers * kJoinRows * kPitch * 4;
    static constexpr bool kQueriesInShared = D == 256;  // 64 registers of queries and 128 of output leave too few
    static constexpr int kQueries = kQueriesInShared ? D / 16 * 512 : 0;  // A operands of all k16 steps, in the order of lanes
    static constexpr int kWeights = kConsumers * kRowTile * (kWarpKeys + 1) * 4;
    static constexpr int kUsed = kQueries + kWeights;    // while keys are read; the join uses the same bytes afterwards
    static constexpr int kBytes = kRing + (kJoin > kUsed ? kJoin : kUsed) + 1024;  // the ring begins at a multiple of 1024
};

__device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kConsumers * 32) : "memory"); }

__device__ __forceinline__ bool consumers_any(bool vote) {
    int any;
    asm volatile(
        "{\n"
        ".reg .pred p, q;\n"
        "setp.ne.s32 p, %1, 0;\n"
        "barrier.cta.red.or.pred q, 1, %2, p;\n"
        "selp.s32 %0, 1, 0, q;\n"
        "}\n"
        : "=r"(any)
        : "r"(static_cast<int>(vote)), "n"(kConsumers * 32)
        : "memory");
    return any != 0;
}

}  // namespace

// T: type of queries and output. Products are of T, or of halves where the cache holds FP8 codes (every code is a half).
template <typename T, int D, bool kCodes>
__global__ void __launch_bounds__(kAttendThreads, AttendSmem<D, kCodes>::kCtas) attend_kernel(const __grid_constant__ AttendDev p) {
    using M = typename std::conditional<kCodes, __half, T>::type;
    using S = Stage<D, kCodes>;
    using Shared = AttendSmem<D, kCodes>;
    constexpr int kStages = Shared::kStages;
    constexpr int kSteps = D / 16;       // k16 steps of q . k
    constexpr int kOut = D / 8;          // n8 tiles of the output
    constexpr int kElem = kCodes ? 1 : 2;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ Pipes<kStages> pipes;
    __shared__ float warp_stats[kConsumers][kRowTile][2];

    const int warp = uniform(static_cast<int>(threadIdx.x >> 5)), lane = threadIdx.x & 31;
    const bool leader = elect_one();
    if (warp == kConsumers && leader) {
        pipes.init(kConsumers, kConsumers);
        tma_prefetch_descriptor(&p.tm_k);
        tma_prefetch_descriptor(&p.tm_v);
    }
    __syncthreads();
    const long long deadline = globaltimer() + kDefaultTimeoutNs;
    pdl_wait();
    pdl_launch_dependents();
    if (warp == kConsumers) {
        produce<kStages, S::kPieces, false>(p, smem, pipes, deadline, leader);
        return;
    }

    // -- the consumers --------------------------------------------------------------------------------------------------
    const int g = lane >> 2, t = lane & 3;
    const S rows_of_stage(min(kTileKeys, 1 << p.page_shift), warp * kWarpKeys);
    int stage = 0, slot = 0;
    uint32_t parity = 0, slot_parity = 0;
    while (true) {
    const bool announced = mbar_wait_warp(&pipes.work_full[slot], slot_parity, deadline);
    if (!announced && leader) stalled(p, 3, slot);
    if (consumers_any(!announced)) return;  // none of the warps may wait for the others any more
    const Work item = pipes.works[slot];
    __syncwarp();
    if (leader) mbar_arrive(&pipes.work_empty[slot]);
    if (++slot == kWorkSlots) slot = 0, slot_parity ^= 1;
    if (item.head < 0) return;
    const int sequence = item.sequence, head = item.head, row_tile = item.row_tile;
    // This thread's two rows: g and g + 8 of the tile.
    const int row0 = row_tile * kRowTile + g, row1 = row0 + 8;
    const int token0 = token_of(p, min(row0, p.rows - 1)), token1 = token_of(p, min(row1, p.rows - 1));
    const int from0 = seen_from(p, item.first_pos, token0), to0 = seen_to(p, item.first_pos, item.length, token0);
    const int from1 = seen_from(p, item.first_pos, token1), to1 = seen_to(p, item.first_pos, item.length, token1);
    const int last_row = min(row_tile * kRowTile + kRowTile, p.rows) - 1;
    const int all_from = seen_from(p, item.first_pos, token_of(p, last_row));                          // from here on every row sees
    const int all_to = seen_to(p, item.first_pos, item.length, token_of(p, row_tile * kRowTile));    // the keys, up to here

    auto q_row = [&](int row) -> const T* {
        const int token = token_of(p, row), of = row - token * p.group;
        return static_cast<const T*>(p.a.q) + sequence * p.a.q_strides[0] + token * p.a.q_strides[1] +
               static_cast<long long>(head * p.group + of) * p.a.q_strides[2];
    };
    // Queries as the A operand. With FP8 keys a lane's elements of a k16 step are four neighbours (see below).
    uint32_t q[kSteps][4];
    const bool has0 = row0 < p.rows, has1 = row1 < p.rows;
    const T* q0 = has0 ? q_row(row0) : nullptr;
    const T* q1 = has1 ? q_row(row1) : nullptr;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
        const int at0 = s * 16 + t * (kCodes ? 4 : 2);
        const int at1 = at0 + (kCodes ? 2 : 8);
        q[s][0] = has0 ? *reinterpret_cast<const uint32_t*>(q0 + at0) : 0;
        q[s][1] = has1 ? *reinterpret_cast<const uint32_t*>(q1 + at0) : 0;
        q[s][2] = has0 ? *reinterpret_cast<const uint32_t*>(q0 + at1) : 0;
        q[s][3] = has1 ? *reinterpret_cast<const uint32_t*>(q1 + at1) : 0;
    }
    float scale0 = p.a.scale * kLog2e, scale1 = scale0;
    if constexpr (kCodes) {
        // A BF16 row may not fit a half: it is scaled by the power of two that brings its largest element below 2 (exact,
        // but for elements 2^-14 of the largest, whose error is at most 2^-25 of it), and the scores are scaled back. (A query
        // as the sum of two E4M3 values, and FP8 products: 170 us against 110 for 24 sequences of 12000 keys, heads of 256.)
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
    const uint32_t* shared_q = nullptr;
    if constexpr (Shared::kQueriesInShared) {
        uint32_t* to = reinterpret_cast<uint32_t*>(smem + Shared::kRing);
        if (warp == 0) {
#pragma unroll
            for (int s = 0; s < kSteps; ++s)
                *reinterpret_cast<uint4*>(to + (s * 32 + lane) * 4) = make_uint4(q[s][0], q[s][1], q[s][2], q[s][3]);
        }
        consumers_sync();
        shared_q = to + lane * 4;
    }

    float o[kOut][4];
#pragma unroll
    for (int i = 0; i < kOut; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;

    for (int tile = 0; tile < item.tiles; ++tile) {
        if (!mbar_wait_warp(&pipes.full[stage], parity, deadline) && leader) stalled(p, 4, tile);
        const int key0 = item.start + tile * kTileKeys + warp * kWarpKeys;
        uint8_t* stage_k = smem + stage * 2 * S::kBytes;
        const uint32_t stage_k32 = smem_u32(stage_k), stage_v32 = stage_k32 + S::kBytes;
        const uint32_t present = static_cast<uint32_t>(pipes.present[stage] >> (warp * kWarpKeys)) & 0xFFFFu;

        auto query_step = [&](int k, uint32_t (&a)[4]) {
            if constexpr (Shared::kQueriesInShared) {
                const uint4 v = *reinterpret_cast<const uint4*>(shared_q + k * 128);
                a[0] = v.x, a[1] = v.y, a[2] = v.z, a[3] = v.w;
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) a[i] = q[k][i];
            }
        };
        // scores: columns are keys, 0..7 in s[0], 8..15 in s[1]
        float s[2][4] = {};
        if constexpr (!kCodes) {
            const int r = (lane & 7) + ((lane >> 4) << 3);
            float more_s[2][4] = {};  // odd steps: half as long a chain of dependent products
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                uint32_t a[4], b[4];
                query_step(k, a);
                ldmatrix_x4(b, stage_k32 + rows_of_stage.at(r, 2 * k + ((lane >> 3) & 1)));
                mma_16816<M>(k & 1 ? more_s[0] : s[0], a, b[0], b[1]);
                mma_16816<M>(k & 1 ? more_s[1] : s[1], a, b[2], b[3]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) s[0][i] += more_s[0][i], s[1][i] += more_s[1][i];
        } else {
            // A 16-byte piece of a key row is one k16 step: lane t of a row holds its elements 4t .. 4t + 3.
            const int r = (lane & 7) + (((lane >> 3) & 1) << 3);
            float more_s[2][4] = {};
#pragma unroll
            for (int k = 0; k < kSteps; k += 2) {
                uint32_t a0[4], a1[4], b[4];
                query_step(k, a0);
                query_step(k + 1, a1);
                ldmatrix_x4(b, stage_k32 + rows_of_stage.at(r, k + (lane >> 4)));
                mma_16816<M>(s[0], a0, e4m3x2_to_f16x2(b[0] & 0xFFFFu), e4m3x2_to_f16x2(b[0] >> 16));
                mma_16816<M>(s[1], a0, e4m3x2_to_f16x2(b[1] & 0xFFFFu), e4m3x2_to_f16x2(b[1] >> 16));
                mma_16816<M>(more_s[0], a1, e4m3x2_to_f16x2(b[2] & 0xFFFFu), e4m3x2_to_f16x2(b[2] >> 16));
                mma_16816<M>(more_s[1], a1, e4m3x2_to_f16x2(b[3] & 0xFFFFu), e4m3x2_to_f16x2(b[3] >> 16));
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) s[0][i] += more_s[0][i], s[1][i] += more_s[1][i];
        }
        const bool by_row = key0 < all_from || key0 + kWarpKeys > all_to;  // rows see different keys of this tile
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

        // Values that are not finite, in a key that some rows see and others do not, or that is not there at all: 0 * inf
        // would reach the result. They are added here to the rows that see them, and are zero in the product below.
        if (by_row || present != 0xFFFFu) {
            // This warp's 16 rows, word by word.
            constexpr int kWords = kWarpKeys * S::kPieces * 4;
            auto word = [&](int i) {
                return reinterpret_cast<uint32_t*>(stage_k + S::kBytes + rows_of_stage.at(i / (S::kPieces * 4), i / 4 % S::kPieces) + i % 4 * 4);
            };
            bool apart = false;
            for (int i = lane; i < kWords; i += 32) apart |= not_finite<M, kCodes>(*word(i)) != 0;
            if (__any_sync(0xFFFFFFFFu, apart)) {
                float* weights = reinterpret_cast<float*>(smem + Shared::kRing + Shared::kQueries);
                float(&w)[kRowTile][kWarpKeys + 1] = reinterpret_cast<float(*)[kRowTile][kWarpKeys + 1]>(weights)[warp];
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    w[g][8 * n + 2 * t] = s[n][0], w[g][8 * n + 2 * t + 1] = s[n][1];
                    w[g + 8][8 * n + 2 * t] = s[n][2], w[g + 8][8 * n + 2 * t + 1] = s[n][3];
                }
                __syncwarp();
#pragma unroll 1
                for (int c = 0; c < kWarpKeys; ++c) {
                    const int key = key0 + c;
                    const bool there = (present >> c) & 1;
                    const bool see0 = there && key >= from0 && key < to0, see1 = there && key >= from1 && key < to1;
                    const float w0 = w[g][c], w1 = w[g + 8][c];
#pragma unroll
                    for (int i = 0; i < kOut; ++i) {
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int byte = (kCodes ? (i / 2) * 16 + 4 * t + 2 * e + (i & 1) : 8 * i + 2 * t + e) * kElem;
                            const uint8_t* at = stage_k + S::kBytes + rows_of_stage.at(c, byte / 16) + byte % 16;
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
                for (int i = lane; i < kWords; i += 32) *word(i) &= ~not_finite<M, kCodes>(*word(i));
                fence_proxy_async();  // these writes come before TMA's next ones
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
                ldmatrix_x4_trans(b, stage_v32 + rows_of_stage.at(r, 2 * i + (lane >> 4)));
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
        __syncwarp();
        if (leader) mbar_arrive(&pipes.empty[stage]);
        if (++stage == kStages) stage = 0, parity ^= 1;
    }

    // -- the four warps' results, a few rows at a time ---------------------------------------------------------------
#pragma unroll
    for (int x = 1; x < 4; x <<= 1) {
        l0 += __shfl_xor_sync(0xFFFFFFFFu, l0, x);
        l1 += __shfl_xor_sync(0xFFFFFFFFu, l1, x);
    }
    if (t == 0) {
        warp_stats[warp][g][0] = m0, warp_stats[warp][g][1] = l0;
        warp_stats[warp][g + 8][0] = m1, warp_stats[warp][g + 8][1] = l1;
    }
    consumers_sync();
    {
        float n0 = -INFINITY, n1 = -INFINITY;
#pragma unroll
        for (int w = 0; w < kConsumers; ++w) n0 = fmaxf(n0, warp_stats[w][g][0]), n1 = fmaxf(n1, warp_stats[w][g + 8][0]);
        // A warp that met no visible key has all zeros, or NaN times zero from a score that was NaN: kept as it is.
        const float f0 = m0 == -INFINITY ? 0.f : exp2_approx(m0 - n0), f1 = m1 == -INFINITY ? 0.f : exp2_approx(m1 - n1);
#pragma unroll
        for (int i = 0; i < kOut; ++i) o[i][0] *= f0, o[i][1] *= f0, o[i][2] *= f1, o[i][3] *= f1;
    }
    const int rows = min(kRowTile, p.rows - row_tile * kRowTile);
    const float value_scale = kCodes ? p.a.cache.v_scale[head] : 1.f;
    float* joined = reinterpret_cast<float*>(smem + Shared::kRing);
    for (int r0 = 0; r0 < rows; r0 += Shared::kJoinRows) {
        if ((g & ~(Shared::kJoinRows - 1)) == (r0 & 7)) {
            float* to = joined + (warp * Shared::kJoinRows + (g & (Shared::kJoinRows - 1))) * Shared::kPitch;
#pragma unroll
            for (int i = 0; i < kOut; ++i) {
                const float x = r0 < 8 ? o[i][0] : o[i][2], y = r0 < 8 ? o[i][1] : o[i][3];
                if constexpr (!kCodes) {
                    *reinterpret_cast<float2*>(to + 8 * i + 2 * t) = make_float2(x, y);
                } else {
                    const int d = (i / 2) * 16 + 4 * t + (i & 1);
                    to[d] = x, to[d + 2] = y;
                }
            }
        }
        consumers_sync();
        for (int i = threadIdx.x; i < min(Shared::kJoinRows, rows - r0) * (D / 4); i += kConsumers * 32) {
            const int r = r0 + i / (D / 4), d = (i % (D / 4)) * 4;
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
            float top = -INFINITY, l = 0.f;
#pragma unroll
            for (int w = 0; w < kConsumers; ++w) {
                const float4 v = *reinterpret_cast<const float4*>(joined + (w * Shared::kJoinRows + (r - r0)) * Shared::kPitch + d);
                sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
                top = fmaxf(top, warp_stats[w][r][0]);
            }
#pragma unroll
            for (int w = 0; w < kConsumers; ++w) {
                const float m = warp_stats[w][r][0];
                l += warp_stats[w][r][1] * (m == -INFINITY ? 0.f : exp2_approx(m - top));
            }
            if (item.whole) {
                finish_row<T>(p, sequence, head, row_tile * kRowTile + r, d, sum, top, l, value_scale);
            } else {
                const int piece = item.piece * p.rows_cap + r;
                *reinterpret_cast<float4*>(p.partial + static_cast<size_t>(piece) * D + d) = sum;
                if (d == 0) *reinterpret_cast<float2*>(p.stats + piece * 2) = make_float2(top, l);
            }
        }
        consumers_sync();
    }
    }
}

// Joins the partial results of an item that lies in several runs (see SplitItem): for each of its rows,
// out = sum_c exp2(m_c - m) o_c / sum_c exp2(m_c - m) l_c. The rows are shared by gridDim.y blocks and their elements by
// gridDim.z; in a block every thread has four elements of a row, and threads that are left over take further partial results
// of the same rows.
constexpr int kJoinMostThreads = 1024;
constexpr int kJoinAhead = 4;  // partial results that a thread has on the way at once

template <typename T, int D>
__global__ void __launch_bounds__(kJoinMostThreads) join_kernel(const __grid_constant__ AttendDev p) {
    extern __shared__ float4 sums[];  // [lines][across], then stats[lines]
    float2* stats = reinterpret_cast<float2*>(sums + blockDim.x);
    const int across = D / 4 / gridDim.z, lines = blockDim.x / across;  // threads along a row, and how often
    const SplitItem item(p, blockIdx.x);
    const int run = item.run, last = item.last, head = item.head, first_row = item.row_tile * kRowTile;
    // Every block waits, those without work too: this kernel's end stands for the end of the one in front.
    pdl_wait();
    pdl_launch_dependents();
    if (!item.split) return;
    const int per_block = (p.rows_cap + gridDim.y - 1) / gridDim.y;
    const int row_begin = blockIdx.y * per_block, row_end = min(min(row_begin + per_block, p.rows_cap), p.rows - first_row);
    const int deep = max(1, lines / per_block);  // threads along the partial results of a row
    const int at = threadIdx.x / across, x = threadIdx.x - at * across + blockIdx.z * across, y = at / per_block;
    const float value_scale = p.a.cache.type == DLM_E4M3 ? p.a.cache.v_scale[head] : 1.f;
    for (int r0 = row_begin; r0 < row_end; r0 += deep == 1 ? lines : per_block) {
        const int r = r0 + (deep == 1 ? at : at % per_block);
        const bool takes_part = r < row_end && (deep == 1 || y < deep);
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        float top = -INFINITY, l = 0.f;
        if (takes_part) {
            for (int c0 = run + (deep == 1 ? 0 : y); c0 <= last; c0 += deep * kJoinAhead) {
                float2 ml[kJoinAhead];
                float4 v[kJoinAhead];
#pragma unroll
                for (int i = 0; i < kJoinAhead; ++i) {
                    const int c = c0 + i * deep;
                    ml[i] = make_float2(-INFINITY, 0.f), v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (c <= last) {
                        const size_t piece = static_cast<size_t>(c * 2 + (c == run)) * p.rows_cap + r;
                        ml[i] = __ldcg(reinterpret_cast<const float2*>(p.stats + piece * 2));
                        v[i] = __ldcg(reinterpret_cast<const float4*>(p.partial + piece * D + x * 4));
                    }
                }
                float n = top;
#pragma unroll
                for (int i = 0; i < kJoinAhead; ++i) n = fmaxf(n, ml[i].x);
                const float keep = top == -INFINITY ? 0.f : exp2_approx(top - n);
                // No visible key so far: zeros, or NaN from a score that was NaN, which stays.
                sum.x *= keep, sum.y *= keep, sum.z *= keep, sum.w *= keep, l *= keep;
                top = n;
#pragma unroll
                for (int i = 0; i < kJoinAhead; ++i) {
                    const float f = ml[i].x == -INFINITY ? 0.f : exp2_approx(ml[i].x - n);
                    l += ml[i].y * f;
                    sum.x += v[i].x * f, sum.y += v[i].y * f, sum.z += v[i].z * f, sum.w += v[i].w * f;
                }
            }
        }
        // The lines of a row are added two by two (the same loop for every thread of the block).
        for (int n = deep; n > 1; n = (n + 1) / 2) {
            const int far = (n + 1) / 2;
            if (takes_part && y >= far && y < n) {
                sums[threadIdx.x] = sum;
                if (threadIdx.x == at * across) stats[at] = make_float2(top, l);
            }
            __syncthreads();
            if (takes_part && y + far < n) {
                const float2 ml = stats[at + far * per_block];
                const float4 v = sums[threadIdx.x + far * per_block * across];
                const float m = fmaxf(top, ml.x);
                const float f = top == -INFINITY ? 0.f : exp2_approx(top - m), h = ml.x == -INFINITY ? 0.f : exp2_approx(ml.x - m);
                top = m, l = l * f + ml.y * h;
                sum.x = sum.x * f + v.x * h, sum.y = sum.y * f + v.y * h, sum.z = sum.z * f + v.z * h, sum.w = sum.w * f + v.w * h;
            }
            __syncthreads();
        }
        if (takes_part && (deep == 1 || y == 0))
            finish_row<T>(p, item.sequence, head, first_row + r, x * 4, sum, top, l, value_scale);
    }
}

template <typename T, int D, bool kCodes>
static int launch_attend_t(const AttendDev& p, const LaunchOpts& o) {
    void* args[] = {const_cast<AttendDev*>(&p)};
    const int rc = launch_kernel<attend_kernel<T, D, kCodes>>(dim3(p.grid), dim3(kAttendThreads), AttendSmem<D, kCodes>::kBytes, args, o);
    if (rc != 0 || p.partial == nullptr) return rc;
    // With fewer items than runs an item may have hundreds of partial results: large blocks, one for a quarter of each row (293
    // partial results of a row: 7 us in blocks of a whole row, all of it latency). Otherwise it has two or three, and most blocks
    // only find out that there is nothing to join (0.5 us; 9000 blocks took 25).
    const long long items = static_cast<long long>(p.a.batch) * p.items;
    const LaunchOpts dependent{o.stream, true, false};  // always a dependent launch of the kernel above
    auto join = [&](unsigned blocks, int rows, int splits, int threads) {
        return launch_kernel<join_kernel<T, D>>(dim3(blocks, rows < 1 ? 1 : rows < p.rows_cap ? rows : p.rows_cap, splits), dim3(threads),
                                                threads * 16 + threads * splits / (D / 4) * 8, args, dependent);
    };
    if (!p.by_item) return join(static_cast<unsigned>(p.grid), 1, 1, 256);
    const int rows = static_cast<int>(p.sms * 2 / items);
    return p.grid > 32 * items ? join(static_cast<unsigned>(items), rows, 4, kJoinMostThreads) : join(static_cast<unsigned>(items), rows, 1, 256);
}

// Calls f with the type and the sizes of a call as compile-time constants.
template <typename F>
static int by_type(int type, int cache_type, int head_dim, F f) {
    auto by_dim = [&](auto t, auto codes) {
        switch (head_dim) {
            case 64: return f(t, std::integral_constant<int, 64>{}, codes);
            case 128: return f(t, std::integral_constant<int, 128>{}, codes);
            default: return f(t, std::integral_constant<int, 256>{}, codes);
        }
    };
    auto by_codes = [&](auto t) { return cache_type == DLM_E4M3 ? by_dim(t, std::true_type{}) : by_dim(t, std::false_type{}); };
    return type == DLM_F16 ? by_codes(__half{}) : by_codes(__nv_bfloat16{});
}

int launch_attend(const AttendDev& p, const LaunchOpts& o) {
    if (p.blocks) return launch_blocks(p, o);
    return by_type(p.a.type, p.a.cache.type, p.a.cache.head_dim, [&](auto t, auto dim, auto codes) {
        return launch_attend_t<decltype(t), decltype(dim)::value, decltype(codes)::value>(p, o);
    });
}

int attend_ctas_per_sm(int type, int cache_type, int head_dim) {
    return by_type(type, cache_type, head_dim,
                   [&](auto, auto dim, auto codes) { return AttendSmem<decltype(dim)::value, decltype(codes)::value>::kCtas; });
}

}  // namespace dlm
