// Attention of new tokens over a paged cache of keys and values (dlmrt/ops/triton/attention.py; split over the keys and
// joined as dlmrt/models/sdar/engine.py:127-132 does).
//
//   o = sum_j exp(s_j) v_j / sum_j exp(s_j),   s_j = scale * q . k_j over the keys that the row's token sees
//
// One pass over the keys with a running reference m and sum l per row (all exponents in base 2, scale * log2(e) folded into the
// scores). What is there is rescaled by exp2(m - m') when a score is more than kRescaleAbove + kHeadroom above m; m' is then the
// new maximum less kHeadroom (see paged_attend.cuh). Weights enter the second product in a high and a low part.
//
// The rows that share a key head are its query heads times the new tokens. 8 or 16 of them are the N of an mma.sync, 16 keys
// (then 16 elements of the output) its M: S^T = K Q^T, O^T = V^T P^T. A single token fills a few rows and is bound by reading
// the cache, so the tensor instructions only have to keep up with HBM; with rows as M half of them or more would be idle.
//
//   warp 4     deals out the work and requests keys and values: steps of 64 keys into a ring of stages, as TMA boxes of a
//              page's slots (pages in any order; up to 64 slots a box). See paged_attend.cuh.
//   warps 0-3  take 16 keys of every step each, with their own maximum, sum and output in registers: no step in which they
//              wait for one another but an item's end, where the four are joined in shared memory.
//
// Many rows (a block of tokens) are another kernel's (paged_blocks.cu).
//
// Bound by HBM: 64 sequences of 129 to 8192 keys, 8 key heads of 128 with four rows each, 88 us, 5.9 TB/s; one sequence of 131071
// keys, 4 heads, 48 us, 5.5 TB/s; FP8, 24 sequences of 1000 to 12000 keys, 8 heads of 256 with two rows, 78 us, 5.7 TB/s, where
// widening the codes takes most of the instructions (114 us with the rows as M of the products).
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

// Shared memory of a CTA, and how many CTAs an SM holds of it (registers are held to what they leave each other). Three of fewer
// stages pay where few registers are needed and a step's latency is long: FP8, 8 rows, heads of 128: 51 us against 54; not for
// 16-bit heads of 128, whose steps need no conversion: 94 against 89.
template <int D, bool kCodes, int kRows>
struct AttendSmem {
    static constexpr bool kThree = D == 64 || (kCodes && kRows == 8);
    static constexpr int kCtas = kThree ? 3 : D == 256 && !kCodes ? 1 : 2;
    static constexpr int kStages = D == 64 ? (kCodes ? 6 : 4) : D == 128 && kCodes ? (kThree ? 4 : 6) : kThree ? 2 : 3;
    static constexpr int kRing = kStages * 2 * Stage<D, kCodes>::kBytes;
    static constexpr int kPitch = D + 4;
    static constexpr int kJoinRows = D == 256 ? 2 : 4;  // rows of a tile that the warps exchange at a time
    static constexpr int kJoin = kConsumers * kJoinRows * kPitch * 4;
    static constexpr bool kQueriesInShared = D == 256;  // 64 registers of queries and 128 of output leave too few
    static constexpr int kQueries = kQueriesInShared ? D * kRows * 2 : 0;  // B operands of all k16 steps, in the order of lanes
    static constexpr int kWeights = kConsumers * kRows * (kWarpKeys + 1) * 4;
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
template <typename T, int D, bool kCodes, int kRows>
__global__ void __launch_bounds__(kAttendThreads, AttendSmem<D, kCodes, kRows>::kCtas) attend_kernel(const __grid_constant__ AttendDev p) {
    using M = typename std::conditional<kCodes, __half, T>::type;
    using S = Stage<D, kCodes>;
    using Shared = AttendSmem<D, kCodes, kRows>;
    constexpr int kStages = Shared::kStages;
    constexpr int kSteps = D / 16;       // k16 steps of q . k
    constexpr int kOut = D / 16;         // m16 tiles of the output
    constexpr int kN = kRows / 8;        // n8 tiles of rows
    constexpr int kChains = 4 / kN;      // sums of products that go on side by side
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ Pipes<kStages> pipes;
    __shared__ float warp_stats[kConsumers][kRows][2];

    const int warp = uniform(static_cast<int>(threadIdx.x >> 5)), lane = threadIdx.x & 31;
    const bool leader = elect_one();
    if (warp == kConsumers && leader) {
        pipes.init(kConsumers, kConsumers);
        tma_prefetch_descriptor(&p.tm_k);
        tma_prefetch_descriptor(&p.tm_v);
    }
    __syncthreads();
    pdl_wait();
    pdl_launch_dependents();
    if (warp == kConsumers) {
        produce<kStages, S::kPieces, false>(p, smem, pipes, leader);
        return;
    }

    // -- the consumers --------------------------------------------------------------------------------------------------
    const int g = lane >> 2, t = lane & 3;
    const S rows_of_stage(min(kTileKeys, 1 << p.page_shift), warp * kWarpKeys);
    int stage = 0, slot = 0;
    uint32_t parity = 0, slot_parity = 0;
    while (true) {
    const long long deadline = item_deadline();
    const bool announced = mbar_wait_warp(&pipes.work_full[slot], slot_parity, deadline);
    if (!announced && leader) stalled(p, 3, slot);
    if (consumers_any(!announced)) return;  // none of the warps may wait for the others any more
    const Work item = pipes.works[slot];
    __syncwarp();
    if (leader) mbar_arrive(&pipes.work_empty[slot]);
    if (++slot == kWorkSlots) slot = 0, slot_parity ^= 1;
    if (item.head < 0) return;
    const int sequence = item.sequence, head = item.head, row_tile = item.row_tile;
    const int first_row = row_tile * kRows, last_row = min(first_row + kRows, p.rows) - 1;
    const int all_from = seen_from(p, item.first_pos, token_of(p, last_row));               // from here on every row sees
    const int all_to = seen_to(p, item.first_pos, item.length, token_of(p, first_row));   // the keys, up to here
    // Keys that a row of the tile sees; this thread has the scores of rows 8 n + 2 t + e.
    auto sees = [&](int row, int* from, int* to) {
        const int token = token_of(p, min(first_row + row, last_row));
        *from = seen_from(p, item.first_pos, token), *to = seen_to(p, item.first_pos, item.length, token);
    };

    auto q_row = [&](int row) -> const T* {
        const int token = token_of(p, row), of = row - token * p.group;
        return static_cast<const T*>(p.a.q) + sequence * p.a.q_strides[0] + token * p.a.q_strides[1] +
               static_cast<long long>(head * p.group + of) * p.a.q_strides[2];
    };
    // Queries as the B operand: row 8 n + g. With FP8 keys a lane's elements of a k16 step are four neighbours (see below).
    uint32_t q[kSteps][kN][2];
    float scale[kN][2];
#pragma unroll
    for (int n = 0; n < kN; ++n) {
        const int row = first_row + 8 * n + g;
        const T* from = row <= last_row ? q_row(row) : nullptr;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const int at = s * 16 + t * (kCodes ? 4 : 2);
            q[s][n][0] = from != nullptr ? *reinterpret_cast<const uint32_t*>(from + at) : 0;
            q[s][n][1] = from != nullptr ? *reinterpret_cast<const uint32_t*>(from + at + (kCodes ? 2 : 8)) : 0;
        }
        scale[n][0] = scale[n][1] = p.a.scale * kLog2e;
        if constexpr (kCodes) {
            // A BF16 row may not fit a half: it is scaled by the power of two that brings its largest element below 2 (exact,
            // but for elements 2^-14 of the largest, whose error is at most 2^-25 of it), and the scores are scaled back. (A
            // query as the sum of two E4M3 values, and FP8 products: 170 us against 110 for 24 sequences of 12000 keys, heads
            // of 256.)
            float top = 0.f;
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                const float2 a = widen2<T>(q[s][n][0]), b = widen2<T>(q[s][n][1]);
                top = fmaxf(fmaxf(top, fmaxf(fabsf(a.x), fabsf(a.y))), fmaxf(fabsf(b.x), fabsf(b.y)));
            }
#pragma unroll
            for (int x = 1; x < 4; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, x));
            // 2^-e and 2^e for the exponent e of the largest element, kept where both are normal numbers.
            const int e = min(max(static_cast<int>(__float_as_uint(top) >> 23) - 127, -126), 126);
            const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23), up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float2 a = widen2<T>(q[s][n][i]);
                    q[s][n][i] = narrow2<__half>(a.x * down, a.y * down);
                }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
                scale[n][i] = scale[n][i] * p.a.cache.k_scale[head] * __shfl_sync(0xFFFFFFFFu, up, (2 * t + i) * 4);
        }
    }
    const uint32_t* shared_q = nullptr;
    if constexpr (Shared::kQueriesInShared) {
        uint32_t* to = reinterpret_cast<uint32_t*>(smem + Shared::kRing);
        if (warp == 0) {
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
#pragma unroll
                for (int n = 0; n < kN; ++n) *reinterpret_cast<uint2*>(to + ((s * kN + n) * 32 + lane) * 2) = make_uint2(q[s][n][0], q[s][n][1]);
            }
        }
        consumers_sync();
        shared_q = to + lane * 2;
    }

    float o[kOut][kN][4];  // [element g of 16 (FP8: 2 g)][row 2 t], [the same][2 t + 1], then element g + 8 (2 g + 1)
    float m[kN][2], l[kN][2];  // l: of this thread's keys
#pragma unroll
    for (int n = 0; n < kN; ++n) {
#pragma unroll
        for (int i = 0; i < kOut; ++i) o[i][n][0] = o[i][n][1] = o[i][n][2] = o[i][n][3] = 0.f;
        m[n][0] = m[n][1] = -INFINITY, l[n][0] = l[n][1] = 0.f;
    }

    for (int tile = 0; tile < item.tiles; ++tile) {
        if (!mbar_wait_warp(&pipes.full[stage], parity, deadline) && leader) stalled(p, 4, tile);
        const int key0 = item.start + tile * kTileKeys + warp * kWarpKeys;
        uint8_t* stage_k = smem + stage * 2 * S::kBytes;
        const uint32_t stage_k32 = smem_u32(stage_k), stage_v32 = stage_k32 + S::kBytes;
        const uint32_t present = static_cast<uint32_t>(pipes.present[stage] >> (warp * kWarpKeys)) & 0xFFFFu;

        auto query_step = [&](int k, int n) {
            if constexpr (Shared::kQueriesInShared) return *reinterpret_cast<const uint2*>(shared_q + (k * kN + n) * 64);
            else return make_uint2(q[k][n][0], q[k][n][1]);
        };
        // scores: [key g][row 2 t], [key g][row 2 t + 1], then key g + 8
        float s[kN][4], sums[kChains][kN][4];
        const int r = lane & 15;
#pragma unroll
        for (int c = 0; c < kChains; ++c) {
#pragma unroll
            for (int n = 0; n < kN; ++n) sums[c][n][0] = sums[c][n][1] = sums[c][n][2] = sums[c][n][3] = 0.f;
        }
        if constexpr (!kCodes) {
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                uint32_t a[4];
                ldmatrix_x4(a, stage_k32 + rows_of_stage.at(r, 2 * k + (lane >> 4)));
#pragma unroll
                for (int n = 0; n < kN; ++n) {
                    const uint2 b = query_step(k, n);
                    mma_16816<M>(sums[k % kChains][n], a, b.x, b.y);
                }
            }
        } else {
            // A 16-byte piece of a key row is one k16 step: lane t of a row holds its elements 4t .. 4t + 3.
#pragma unroll
            for (int k = 0; k < kSteps; k += 2) {
                uint32_t w[4];
                ldmatrix_x4(w, stage_k32 + rows_of_stage.at(r, k + (lane >> 4)));
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const uint32_t a[4] = {e4m3x2_to_f16x2(w[2 * c] & 0xFFFFu), e4m3x2_to_f16x2(w[2 * c + 1] & 0xFFFFu),
                                           e4m3x2_to_f16x2(w[2 * c] >> 16), e4m3x2_to_f16x2(w[2 * c + 1] >> 16)};
#pragma unroll
                    for (int n = 0; n < kN; ++n) {
                        const uint2 b = query_step(k + c, n);
                        mma_16816<M>(sums[(k + c) % kChains][n], a, b.x, b.y);
                    }
                }
            }
        }
#pragma unroll
        for (int n = 0; n < kN; ++n) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (kChains == 4) s[n][e] = (sums[0][n][e] + sums[1][n][e]) + (sums[2][n][e] + sums[3][n][e]);
                else s[n][e] = sums[0][n][e] + sums[1][n][e];
                s[n][e] *= scale[n][e & 1];
            }
        }
        const bool by_row = key0 < all_from || key0 + kWarpKeys > all_to;  // rows see different keys of this tile
        if (by_row || present != 0xFFFFu) {
#pragma unroll
            for (int n = 0; n < kN; ++n) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    int from, to;
                    sees(8 * n + 2 * t + e, &from, &to);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int c = g + 8 * h, key = key0 + c;
                        if (!(present >> c & 1) || key < from || key >= to) s[n][2 * h + e] = -INFINITY;
                    }
                }
            }
        }
        bool rescale = false;
#pragma unroll
        for (int n = 0; n < kN; ++n) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float top = fmaxf(s[n][e], s[n][2 + e]);
                rescale |= top > m[n][e] + (kRescaleAbove + kHeadroom<M>) || (m[n][e] == -INFINITY && top > m[n][e]);
            }
        }
        if (__any_sync(0xFFFFFFFFu, rescale)) {
#pragma unroll
            for (int n = 0; n < kN; ++n) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float top = fmaxf(s[n][e], s[n][2 + e]);
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, x));
                    const float now = fmaxf(m[n][e], top - kHeadroom<M>), f = m[n][e] == now ? 1.f : exp2_approx(m[n][e] - now);
                    m[n][e] = now, l[n][e] *= f;
#pragma unroll
                    for (int i = 0; i < kOut; ++i) o[i][n][e] *= f, o[i][n][2 + e] *= f;
                }
            }
        }
#pragma unroll
        for (int n = 0; n < kN; ++n) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float sub = m[n][e] == -INFINITY ? 0.f : m[n][e];
                s[n][e] = exp2_approx(s[n][e] - sub), s[n][2 + e] = exp2_approx(s[n][2 + e] - sub);
                l[n][e] += s[n][e] + s[n][2 + e];
            }
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
                float(&w)[kRows][kWarpKeys + 1] = reinterpret_cast<float(*)[kRows][kWarpKeys + 1]>(weights)[warp];
#pragma unroll
                for (int n = 0; n < kN; ++n) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[8 * n + 2 * t + (e & 1)][g + 8 * (e >> 1)] = s[n][e];
                }
                __syncwarp();
#pragma unroll 1
                for (int c = 0; c < kWarpKeys; ++c) {
                    const int key = key0 + c;
                    float weight[kN][2];
                    bool see[kN][2];
#pragma unroll
                    for (int n = 0; n < kN; ++n) {
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            int from, to;
                            sees(8 * n + 2 * t + e, &from, &to);
                            see[n][e] = (present >> c & 1) && key >= from && key < to;
                            weight[n][e] = w[8 * n + 2 * t + e][c];
                        }
                    }
#pragma unroll
                    for (int i = 0; i < kOut; ++i) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int byte = kCodes ? 16 * i + 2 * g + h : (16 * i + g + 8 * h) * 2;
                            const uint8_t* at = stage_k + S::kBytes + rows_of_stage.at(c, byte / 16) + byte % 16;
                            float v;
                            if constexpr (kCodes) v = widen2<__half>(e4m3x2_to_f16x2(*at)).x;
                            else v = widen2<M>(*reinterpret_cast<const uint16_t*>(at)).x;
                            if (!isfinite(v)) {
#pragma unroll
                                for (int n = 0; n < kN; ++n) {
#pragma unroll
                                    for (int e = 0; e < 2; ++e)
                                        if (see[n][e]) o[i][n][2 * h + e] += weight[n][e] * v;
                                }
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
            uint32_t b[kN][2], low[kN][2];  // the weights, high and low parts, rows from key g to row g
#pragma unroll
            for (int n = 0; n < kN; ++n) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    split_weights<M, kCodes>(s[n][2 * h], s[n][2 * h + 1], &b[n][h], &low[n][h]);
                    b[n][h] = transpose_8x8(b[n][h]), low[n][h] = transpose_8x8(low[n][h]);
                }
            }
            if constexpr (!kCodes) {
                const int key = (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
                for (int i = 0; i < kOut; ++i) {
                    uint32_t a[4];
                    ldmatrix_x4_trans(a, stage_v32 + rows_of_stage.at(key, 2 * i + ((lane >> 3) & 1)));
#pragma unroll
                    for (int n = 0; n < kN; ++n) mma_16816<M>(o[i][n], a, low[n][0], low[n][1]);
#pragma unroll
                    for (int n = 0; n < kN; ++n) mma_16816<M>(o[i][n], a, b[n][0], b[n][1]);
                }
            } else {
                // w[0], w[1]: keys 2t, 2t + 1 (+ 8) of elements 2g and 2g + 1 of a 16-byte piece; w[2], w[3]: the next piece. The
                // even elements are the product's first eight rows, the odd ones its last.
#pragma unroll
                for (int i = 0; i < kOut; i += 2) {
                    uint32_t w[4];
                    ldmatrix_x4_trans(w, stage_v32 + rows_of_stage.at(r, i + (lane >> 4)));
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const uint32_t a[4] = {
                            e4m3x2_to_f16x2(__byte_perm(w[2 * c], 0, 0x4420)), e4m3x2_to_f16x2(__byte_perm(w[2 * c], 0, 0x4431)),
                            e4m3x2_to_f16x2(__byte_perm(w[2 * c + 1], 0, 0x4420)), e4m3x2_to_f16x2(__byte_perm(w[2 * c + 1], 0, 0x4431))};
#pragma unroll
                        for (int n = 0; n < kN; ++n) mma_16816<M>(o[i + c][n], a, low[n][0], low[n][1]);
#pragma unroll
                        for (int n = 0; n < kN; ++n) mma_16816<M>(o[i + c][n], a, b[n][0], b[n][1]);
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
    for (int n = 0; n < kN; ++n) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) l[n][e] += __shfl_xor_sync(0xFFFFFFFFu, l[n][e], x);
            if (g == 0) warp_stats[warp][8 * n + 2 * t + e][0] = m[n][e], warp_stats[warp][8 * n + 2 * t + e][1] = l[n][e];
        }
    }
    consumers_sync();
#pragma unroll
    for (int n = 0; n < kN; ++n) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < kConsumers; ++w) top = fmaxf(top, warp_stats[w][8 * n + 2 * t + e][0]);
            // A warp that met no visible key has all zeros, or NaN times zero from a score that was NaN: kept as it is.
            const float f = m[n][e] == -INFINITY ? 0.f : exp2_approx(m[n][e] - top);
#pragma unroll
            for (int i = 0; i < kOut; ++i) o[i][n][e] *= f, o[i][n][2 + e] *= f;
        }
    }
    const int rows = last_row + 1 - first_row;
    const float value_scale = kCodes ? p.a.cache.v_scale[head] : 1.f;
    float* joined = reinterpret_cast<float*>(smem + Shared::kRing);
    for (int r0 = 0; r0 < rows; r0 += Shared::kJoinRows) {
        if ((2 * t & ~(Shared::kJoinRows - 1)) == (r0 & 7)) {
            float* to = joined + (warp * Shared::kJoinRows + (2 * t & (Shared::kJoinRows - 1))) * Shared::kPitch;
#pragma unroll
            for (int i = 0; i < kOut; ++i) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int d = 16 * i + (kCodes ? 2 * g + (e >> 1) : g + 8 * (e >> 1));
                    to[(e & 1) * Shared::kPitch + d] = r0 < 8 ? o[i][0][e] : o[i][kN - 1][e];
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
                finish_row<T>(p, sequence, head, first_row + r, d, sum, top, l, value_scale);
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
    const int run = item.run, last = item.last, head = item.head, first_row = item.row_tile * p.tile_rows;
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

template <typename T, int D, bool kCodes, int kRows>
static int launch_attend_t(const AttendDev& p, const LaunchOpts& o) {
    void* args[] = {const_cast<AttendDev*>(&p)};
    const int rc = launch_kernel<attend_kernel<T, D, kCodes, kRows>>(dim3(p.grid), dim3(kAttendThreads), AttendSmem<D, kCodes, kRows>::kBytes, args, o);
    if (rc != 0 || p.partial == nullptr) return rc;
    // With far fewer items than runs an item has many partial results: large blocks, one for a quarter of each row (four items in
    // 296 runs, 131071 keys: 48.6 us in all, 49.5 with small blocks; 18 items in 444 runs: 18.2 against 12.1). Otherwise it has
    // two or three, and most blocks only find out that there is nothing to join (0.5 us; 9000 blocks took 25).
    const long long items = static_cast<long long>(p.a.batch) * p.items;
    const LaunchOpts dependent{o.stream, true, false};  // always a dependent launch of the kernel above
    auto join = [&](unsigned blocks, int rows, int splits, int threads) {
        return launch_kernel<join_kernel<T, D>>(dim3(blocks, rows < 1 ? 1 : rows < p.rows_cap ? rows : p.rows_cap, splits), dim3(threads),
                                                threads * 16 + threads * splits / (D / 4) * 8, args, dependent);
    };
    if (!p.by_item) return join(static_cast<unsigned>(p.grid), 1, 1, 256);
    const bool deep = p.grid > 64 * items;
    const int splits = deep ? 4 : 1, rows = static_cast<int>(p.sms * 2 / (items * splits));  // two blocks an SM
    return join(static_cast<unsigned>(items), rows, splits, deep ? kJoinMostThreads : 256);
}

// Calls f with the type and the sizes of a call as compile-time constants.
template <typename F>
static int by_type(int type, int cache_type, int head_dim, int tile_rows, F f) {
    auto by_rows = [&](auto t, auto codes, auto dim) {
        return tile_rows == kFewRows ? f(t, dim, codes, std::integral_constant<int, kFewRows>{}) : f(t, dim, codes, std::integral_constant<int, kRowTile>{});
    };
    auto by_dim = [&](auto t, auto codes) {
        switch (head_dim) {
            case 64: return by_rows(t, codes, std::integral_constant<int, 64>{});
            case 128: return by_rows(t, codes, std::integral_constant<int, 128>{});
            default: return by_rows(t, codes, std::integral_constant<int, 256>{});
        }
    };
    auto by_codes = [&](auto t) { return cache_type == DLM_E4M3 ? by_dim(t, std::true_type{}) : by_dim(t, std::false_type{}); };
    return type == DLM_F16 ? by_codes(__half{}) : by_codes(__nv_bfloat16{});
}

int launch_attend(const AttendDev& p, const LaunchOpts& o) {
    if (p.blocks) return launch_blocks(p, o);
    return by_type(p.a.type, p.a.cache.type, p.a.cache.head_dim, p.tile_rows, [&](auto t, auto dim, auto codes, auto rows) {
        return launch_attend_t<decltype(t), decltype(dim)::value, decltype(codes)::value, decltype(rows)::value>(p, o);
    });
}

int attend_ctas_per_sm(int type, int cache_type, int head_dim, int tile_rows) {
    return by_type(type, cache_type, head_dim, tile_rows, [&](auto, auto dim, auto codes, auto rows) {
        return AttendSmem<decltype(dim)::value, decltype(codes)::value, decltype(rows)::value>::kCtas;
    });
}

}  // namespace dlm
