// Attention over the paged cache for blocks of tokens: more rows share a key head's keys than a warp's tile holds (a block of
// 32 tokens of four query heads each is 128), so that a step's arithmetic is worth a 128-row tile in tensor memory.
//
//   softmax    groups of four warps, a row of the tile each thread: Q into shared memory, then for every step of 64 keys the row
//              of scores out of tensor memory, mask, maximum, weights exp2(s - m) back into tensor memory over the scores, and
//              their sum. Two groups take steps in turn, each with its own maximum, sum and O, and put them together at an
//              item's end (heads of 256 leave tensor memory for one).
//   producer   a warp, see paged_attend.cuh.
//   converters (FP8 cache) warps that widen a step's codes to halves, exactly, and lay them out as TMA lays out 16-bit keys and
//              values. Queries are halves, too, each row scaled by a power of two.
//   issuer     a warp that issues S = Q K^T (M = 128 rows, N = 64 keys) and O += P V (M = 128, N = head_dim; P from tensor memory in
//              a high and a low part, V as it lies, its 64 keys down the rows). Each group has two buffers of S: its next step's
//              scores are computed under this one's softmax.
//
// m is the reference that weights are relative to when O was last rescaled (see paged_attend.cuh): O, which lives in tensor memory, is
// multiplied by exp2(m - m') only when some row's maximum is more than kRescaleAbove + kHeadroom past m.
//
// One CTA an SM; shared memory holds 2 to 8 steps of 64 keys. A step is 3 * 128 * 64 * head_dim multiply-adds (768 cycles of the
// tensor pipe at 128) and 8192 exponentials (512 cycles). A group took 1300 cycles for a step when weights had one part, most of it
// latency, which is as long as a step's 32 KB take from HBM: with one group nothing would be left to catch up with what an item's
// beginning and end cost. 16 sequences of 1056 to 8224 keys, blocks of 32 tokens, 8 key heads of 128 with four query heads
// each: 63 us, 3.8 TB/s (start 4.5 us, 3.5 between items, join 3); the same over an FP8 cache 83 us, the converters' two warps being
// what takes longest.
#include "paged_attend.cuh"

namespace dlm {

namespace {

constexpr int kGroupThreads = 128;

template <int D, bool kCodes>
struct BlockShape {
    static constexpr int kGroups = D == 256 ? 1 : 2;
    static constexpr int kBuffers = 2 * kGroups;              // of S
    static constexpr int kProducerWarp = 4 * kGroups, kIssuerWarp = kProducerWarp + 1;
    static constexpr int kConverters = !kCodes ? 0 : D == 256 ? 4 : 2;  // 12 warps leave the softmax its 168 registers
    static constexpr int kThreads = kGroups * kGroupThreads + 64 + kConverters * 32;
    static constexpr int kSteps = D == 256 ? 2 : kCodes ? (D == 128 ? 3 : 6) : D == 128 ? 5 : 8;  // whose operands are there
    static constexpr int kStages = !kCodes ? kSteps : D == 256 ? 1 : D == 128 ? 5 : 8;             // of what TMA brings
    static constexpr int kBytes = kTileKeys * D * 2;          // keys, or values, of a step
    static constexpr int kCodeBytes = kTileKeys * D;
    static constexpr int kSteady = kSteps * 2 * kBytes;
    static constexpr int kQueries = kBlockRows * D * 2;
    static constexpr int kRing = kSteady + kQueries;          // where stages of codes begin
    static constexpr int kAll = kRing + (kCodes ? kStages * 2 * kCodeBytes : 0) + 1024;  // it begins at a multiple of 1024
    static constexpr uint32_t kColumns = 512;                 // of tensor memory: an O of each group, then the buffers of S
};

// Instruction descriptor of kind::f16, see umma_idesc_bf16: T is BF16 or FP16, B is K-major, or MN-major where `b_mn`.
template <typename T>
__device__ __forceinline__ constexpr uint32_t idesc_f16(int m, int n, bool b_mn) {
    const uint32_t format = std::is_same<T, __half>::value ? 0 : 1;
    return (1u << 4) | (format << 7) | (format << 10) | (static_cast<uint32_t>(b_mn) << 16) | (static_cast<uint32_t>(n >> 3) << 17) |
           (static_cast<uint32_t>(m >> 4) << 24);
}

// Descriptor of an MN-major operand under the 128-byte swizzle: rows of 64 elements along N, 8 k's a group of 1024 bytes;
// `blocks` bytes from one 64 elements of N to the next.
__device__ __forceinline__ uint64_t umma_desc_mn128(uint32_t smem, uint32_t blocks) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((smem & 0x3FFFF) >> 4);
    d |= static_cast<uint64_t>(blocks >> 4) << 16;
    d |= static_cast<uint64_t>(1024 >> 4) << 32;
    d |= static_cast<uint64_t>(1) << 46;
    d |= static_cast<uint64_t>(2) << 61;
    return d;
}

// D[tmem] += A[tmem] * B[smem], A being 128 rows of 16 k's in 8 columns of 16-bit pairs.
__device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc) {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, 1, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
        "}\n"
        ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc)
        : "memory");
}

__device__ __forceinline__ void tmem_load_32(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_store_32(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
          "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]),
          "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]),
          "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// The warps that share 32 rows, one of each group, meet.
template <int kGroups>
__device__ __forceinline__ void rows_sync(int quarter) {
    if constexpr (kGroups > 1) {
        tcgen05_fence_before();
        asm volatile("bar.sync %0, %1;" ::"r"(quarter + 1), "n"(kGroups * 32) : "memory");
        tcgen05_fence_after();
    }
}
template <int kThreads>
__device__ __forceinline__ bool any_of(int barrier, bool vote) {
    int any;
    asm volatile(
        "{\n"
        ".reg .pred p, q;\n"
        "setp.ne.s32 p, %1, 0;\n"
        "barrier.cta.red.or.pred q, %2, %3, p;\n"
        "selp.s32 %0, 1, 0, q;\n"
        "}\n"
        : "=r"(any)
        : "r"(static_cast<int>(vote)), "r"(barrier), "n"(kThreads)
        : "memory");
    return any != 0;
}
template <int kGroups>
__device__ __forceinline__ bool rows_any(int quarter, bool vote) {
    if constexpr (kGroups == 1) return __any_sync(0xFFFFFFFFu, vote);
    return any_of<kGroups * 32>(quarter + 1, vote);
}
// The warps of a group meet.
__device__ __forceinline__ bool group_any(int group, bool vote) { return any_of<kGroupThreads>(group + 5, vote); }

// 16-byte piece `c` of row `r` of a tile of 128 rows, in column blocks of 128 bytes under the 128-byte swizzle.
__device__ __forceinline__ uint4* tile_piece(uint8_t* tile, int r, int c) {
    return reinterpret_cast<uint4*>(tile + (c / 8) * (kBlockRows * 128) + r * 128 + ((c % 8) ^ (r & 7)) * 16);
}

// Goes through 32 rows of D 16-bit elements, D / 8 lanes of 16 bytes each: every lane passes the address of its own row. One of
// kWays warps that share the rows takes `part`. f(turn, row, piece, address).
template <int D, int kWays, typename F>
__device__ __forceinline__ void by_rows(const void* mine, int part, F f) {
    constexpr int kAcross = D / 8, kAtOnce = 32 / kAcross, kTurns = 32 / kAtOnce / kWays;
    const int lane = threadIdx.x & 31;
    const unsigned long long at = reinterpret_cast<unsigned long long>(mine);
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
        const int r = (i * kWays + part) * kAtOnce + lane / kAcross;
        f(i, r, lane % kAcross, reinterpret_cast<uint8_t*>(__shfl_sync(0xFFFFFFFFu, at, r)));
    }
}

// All-ones in the 16-bit halves of a word that are infinite or NaN.
template <typename T>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
    constexpr uint32_t kExponent = std::is_same<T, __half>::value ? 0x7C007C00u : 0x7F807F80u;
    return __vcmpeq2(w & kExponent, kExponent);
}

// 8 elements of a row, the rest of which kLanes neighbouring lanes have, to halves: scaled by the power of two that brings the
// row's largest element below 2 (see attend_kernel). Returns what undoes it.
template <typename T, int kLanes>
__device__ __forceinline__ float to_halves(uint4* v) {
    uint32_t(&w)[4] = reinterpret_cast<uint32_t(&)[4]>(*v);
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 x = widen2<T>(w[i]);
        top = fmaxf(top, fmaxf(fabsf(x.x), fabsf(x.y)));
    }
#pragma unroll
    for (int x = 1; x < kLanes; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, x));
    const int e = min(max(static_cast<int>(__float_as_uint(top) >> 23) - 127, -126), 126);
    const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 x = widen2<T>(w[i]);
        w[i] = narrow2<__half>(x.x * down, x.y * down);
    }
    return __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
}

}  // namespace

// T: type of queries and output. Products are of T, or of halves where the cache holds FP8 codes.
template <typename T, int D, bool kCodes>
__global__ void __launch_bounds__(BlockShape<D, kCodes>::kThreads, 1) blocks_kernel(const __grid_constant__ AttendDev p) {
    using Shape = BlockShape<D, kCodes>;
    using M = typename std::conditional<kCodes, __half, T>::type;
    constexpr int kStages = Shape::kStages, kSteps = Shape::kSteps, kBytes = Shape::kBytes, kGroups = Shape::kGroups, kBuffers = Shape::kBuffers;
    constexpr int kBlockBytes = kTileKeys * 128;  // 64 keys of a column block of 64 elements
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* queries = smem + Shape::kSteady;
    __shared__ Pipes<kStages> pipes;
    // Queries written; of the step that a buffer of S is for: scores computed, weights written, values consumed; a side step of
    // a group. A wait can only tell a phase from the one before it, which here is kBuffers steps back.
    __shared__ uint64_t q_full, s_full[kBuffers], p_full[kBuffers], pv_done[kBuffers], aside[kGroups];
    __shared__ uint64_t drained;  // what the issuer has on the way, where a wait of its ran out
    // FP8: what the producer's barriers are to the converters, these are to the issuer.
    __shared__ uint64_t wide_full[kSteps], wide_empty[kSteps], wide_present[kSteps];
    uint64_t* const step_full = kCodes ? wide_full : pipes.full;
    uint64_t* const step_empty = kCodes ? wide_empty : pipes.empty;
    uint64_t* const step_present = kCodes ? wide_present : pipes.present;
    __shared__ uint32_t tmem_base;
    __shared__ float row_scale[kCodes ? kBlockRows : 1];
    __shared__ float2 group_stats[kGroups][kBlockRows];  // maximum and sum of a group's steps

    const int warp = uniform(static_cast<int>(threadIdx.x >> 5)), lane = threadIdx.x & 31;
    const bool leader = elect_one();
    if (warp == Shape::kProducerWarp && leader) {
        pipes.init(kCodes ? Shape::kConverters : 1, kGroups * 4 + 1 + Shape::kConverters);
        if constexpr (kCodes)
            for (int i = 0; i < kSteps; ++i) mbar_init(&wide_full[i], Shape::kConverters), mbar_init(&wide_empty[i], 1);
        mbar_init(&q_full, kGroups * kGroupThreads);
        for (int i = 0; i < kBuffers; ++i) mbar_init(&s_full[i], 1), mbar_init(&p_full[i], kGroupThreads), mbar_init(&pv_done[i], 1);
        for (int i = 0; i < kGroups; ++i) mbar_init(&aside[i], kGroupThreads);
        mbar_init(&drained, 1);
        fence_barrier_init();
        tma_prefetch_descriptor(&p.tm_k);
        tma_prefetch_descriptor(&p.tm_v);
    }
    if (warp == Shape::kIssuerWarp) tmem_alloc(&tmem_base, Shape::kColumns);
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem = uniform(tmem_base);
    const uint32_t tmem_s = tmem + kGroups * D;  // S of step n: + (n % kBuffers) * 64; its weights take the place, high parts, then low ones
    auto buffer = [](uint32_t step) { return step % kBuffers; };
    auto phase = [](uint32_t step) { return step / kBuffers & 1; };
    pdl_wait();
    pdl_launch_dependents();

    if (warp == Shape::kProducerWarp) {
        if constexpr (kCodes) produce<kStages, D / 16, true>(p, smem + Shape::kRing, pipes, leader);
        else produce<kStages, D / 8, true>(p, smem, pipes, leader);
    } else if (warp == Shape::kIssuerWarp) {
        // -- the issuer: a whole warp on uniform values, one lane issuing ------------------------------------------------
        constexpr uint32_t kIdescS = idesc_f16<M>(kBlockRows, kTileKeys, false), kIdescO = idesc_f16<M>(kBlockRows, D, true);
        const uint64_t q_desc = umma_desc_k128(queries);
        int stage = 0, slot = 0, next_stage = 0;
        uint32_t parity = 0, slot_parity = 0, q_parity = 0, step = 0;
        long long deadline = 0;
        bool failed = false;
        auto wait = [&](uint64_t* bar, uint32_t bar_phase, int who, int at) {
            if (!mbar_wait_warp(bar, bar_phase, deadline)) {
                failed = true;
                if (leader) stalled(p, who, at);
            }
            tcgen05_fence_after();
        };
        while (true) {
            deadline = item_deadline();
            const bool announced = mbar_wait_warp(&pipes.work_full[slot], slot_parity, deadline);
            if (!announced) {
                failed = true;
                if (leader) stalled(p, 5, slot);
                break;
            }
            const int head = pipes.works[slot].head, tiles = pipes.works[slot].tiles;
            __syncwarp();
            if (leader) mbar_arrive(&pipes.work_empty[slot]);
            if (++slot == kWorkSlots) slot = 0, slot_parity ^= 1;
            if (head < 0) break;
            if (tiles == 0) continue;  // nothing to compute, and no queries were brought
            wait(&q_full, q_parity, 6, tiles);
            q_parity ^= 1;
            auto scores = [&](uint32_t n) {  // of step n, whose keys are the next stage's
                wait(&step_full[next_stage], parity, 7, n);
                const uint32_t keys = smem_u32(smem) + next_stage * 2 * kBytes;
                const uint64_t k_desc = (q_desc & 0xFFFFFFFF00000000ull) | (umma_desc_k128(smem) & 0xFFFF0000u) | ((keys & 0x3FFFF) >> 4);
                if (leader) {
#pragma unroll
                    for (int k = 0; k < D / 16; ++k)
                        umma_bf16(tmem_s + buffer(n) * 64, q_desc + (k / 4) * (kBlockRows * 128 >> 4) + (k % 4) * 2,
                                  k_desc + (k / 4) * (kBlockBytes >> 4) + (k % 4) * 2, kIdescS, k != 0);
                    umma_commit(&s_full[buffer(n)]);
                }
                if (++next_stage == kSteps) next_stage = 0, parity ^= 1;
            };
            for (int ahead = 0; ahead < kGroups && ahead < tiles; ++ahead) scores(step + ahead);
            for (int tile = 0; tile < tiles; ++tile, ++step) {
                if (tile + kGroups < tiles) {
                    // The buffer held the weights of the group's step before, which have to have been consumed.
                    const uint32_t next = step + kGroups;
                    if (tile >= kGroups) wait(&pv_done[buffer(next - kBuffers)], phase(next - kBuffers), 8, tile);
                    scores(next);
                }
                wait(&p_full[buffer(step)], phase(step), 9, tile);
                const uint32_t values = smem_u32(smem) + stage * 2 * kBytes + kBytes;
                if (leader) {
#pragma unroll
                    for (int k = 0; k < kTileKeys / 16; ++k) {
                        const uint64_t v_desc = umma_desc_mn128(values + k * 2048, kBlockBytes);
                        umma_f16_ts(tmem + step % kGroups * D, tmem_s + buffer(step) * 64 + k * 8, v_desc, kIdescO);
                        umma_f16_ts(tmem + step % kGroups * D, tmem_s + buffer(step) * 64 + 32 + k * 8, v_desc, kIdescO);
                    }
                    umma_commit(&step_empty[stage]);
                    umma_commit(&pv_done[buffer(step)]);
                }
                if (++stage == kSteps) stage = 0;
            }
        }
        if (failed) {  // products still read shared memory and write tensor memory, which the block is about to give back
            if (leader) umma_commit(&drained);
            mbar_wait_warp(&drained, 0, globaltimer() + kDrainNs);
        }
    } else if (kCodes && warp > Shape::kIssuerWarp) {
        // -- the converters: pieces of 16 codes ------------------------------------------------------------------------------
        // Eight lanes take four pieces of two keys k and k ^ 5, which puts both their reads and their writes (every other piece of
        // a row) on different banks. A turn goes on by a multiple of 8 keys, under the same swizzle, then by four pieces.
        constexpr int kPieces = D / 16, kRowBytes = kPieces < 8 ? D : 128;
        constexpr int kKeysATurn = 8 * (kCodes ? Shape::kConverters : 1), kTurns = kTileKeys * (kPieces / 4) / kKeysATurn;
        const int part = warp - Shape::kIssuerWarp - 1, key0 = (part * 8 + (lane >> 3) * 2) ^ (lane & 4 ? 5 : 0);
        const int first_code = key0 * kRowBytes + ((lane & 3) ^ (kPieces < 8 ? (key0 >> 1) & 3 : key0 & 7)) * 16;
        const int first_wide = key0 * 128 + (((lane & 3) * 2) ^ (key0 & 7)) * 16;
        int stage = 0, step = 0, slot = 0;
        uint32_t parity = 0, step_parity = 1, slot_parity = 0;
        long long deadline = 0;
        while (true) {
            deadline = item_deadline();
            const bool announced = mbar_wait_warp(&pipes.work_full[slot], slot_parity, deadline);
            if (!announced) {
                if (leader) stalled(p, 16, slot);
                break;
            }
            const int head = pipes.works[slot].head, tiles = pipes.works[slot].tiles;
            __syncwarp();
            if (leader) mbar_arrive(&pipes.work_empty[slot]);
            if (++slot == kWorkSlots) slot = 0, slot_parity ^= 1;
            if (head < 0) break;
            for (int tile = 0; tile < tiles; ++tile) {
                if (!mbar_wait_warp(&pipes.full[stage], parity, deadline) && leader) stalled(p, 17, tile);
                if (!mbar_wait_warp(&wide_empty[step], step_parity, deadline) && leader) stalled(p, 18, tile);
                const uint8_t* codes = smem + Shape::kRing + stage * 2 * Shape::kCodeBytes;
                uint8_t* wide = smem + step * 2 * kBytes;
#pragma unroll 1
                for (int i = 0; i < 2; ++i) {  // keys, values
                    const uint8_t* from = codes + i * Shape::kCodeBytes;
                    uint8_t* to = wide + i * kBytes;
                    uint4 v[kTurns];
#pragma unroll
                    for (int j = 0; j < kTurns; ++j) {
                        const int key = j * kKeysATurn % kTileKeys, c = j * kKeysATurn / kTileKeys;  // from the first turn's
                        v[j] = *reinterpret_cast<const uint4*>(from + (first_code ^ (c % 2 * 64)) + c / 2 * kBlockBytes + key * kRowBytes);
                    }
#pragma unroll
                    for (int j = 0; j < kTurns; ++j) {
                        const int key = j * kKeysATurn % kTileKeys, c = j * kKeysATurn / kTileKeys;
                        auto pair = [&](uint32_t a, uint32_t b) {
                            return make_uint4(e4m3x2_to_f16x2(a & 0xFFFFu), e4m3x2_to_f16x2(a >> 16), e4m3x2_to_f16x2(b & 0xFFFFu),
                                              e4m3x2_to_f16x2(b >> 16));
                        };
                        *reinterpret_cast<uint4*>(to + first_wide + c * kBlockBytes + key * 128) = pair(v[j].x, v[j].y);
                        *reinterpret_cast<uint4*>(to + (first_wide ^ 16) + c * kBlockBytes + key * 128) = pair(v[j].z, v[j].w);
                    }
                }
                if (leader && part == 0) wide_present[step] = pipes.present[stage];
                fence_proxy_async();
                __syncwarp();
                if (leader) mbar_arrive(&wide_full[step]), mbar_arrive(&pipes.empty[stage]);
                if (++stage == kStages) stage = 0, parity ^= 1;
                if (++step == kSteps) step = 0, step_parity ^= 1;
            }
        }
    } else {
        // -- a row of the tile each thread, every kGroups-th step ------------------------------------------------------------
        const int quarter = warp & 3, group = warp >> 2, r = quarter * 32 + lane;
        const uint32_t mine = static_cast<uint32_t>(quarter * 32) << 16;  // this warp's lanes of tensor memory
        const uint32_t tmem_o = tmem + mine + group * D;
        int stage = 0, slot = 0;
        uint32_t slot_parity = 0, step = 0, aside_parity = 0;
        long long deadline = 0;
        auto wait = [&](uint64_t* bar, uint32_t bar_phase, int who, int at) {
            if (!mbar_wait(bar, bar_phase, deadline)) stalled(p, who, at);
            __syncwarp();
            tcgen05_fence_after();
        };
        while (true) {
            deadline = item_deadline();
            const bool announced = mbar_wait_warp(&pipes.work_full[slot], slot_parity, deadline);
            if (!announced && leader) stalled(p, 10, slot);
            if (rows_any<kGroups>(quarter, !announced)) break;  // neither may wait for the other any more
            const Work item = pipes.works[slot];
            __syncwarp();
            if (leader) mbar_arrive(&pipes.work_empty[slot]);
            if (++slot == kWorkSlots) slot = 0, slot_parity ^= 1;
            if (item.head < 0) break;
            const int first_row = item.row_tile * kBlockRows, row = first_row + r, last_row = min(first_row + kBlockRows, p.rows) - 1;
            const int token = token_of(p, min(row, last_row));
            const int from = seen_from(p, item.first_pos, token), to = seen_to(p, item.first_pos, item.length, token);
            const int all_from = seen_from(p, item.first_pos, token_of(p, last_row));                     // from here on every row sees
            const int all_to = seen_to(p, item.first_pos, item.length, token_of(p, first_row));         // the keys, up to here
            const int query_head = item.head * p.group + min(row, last_row) - token * p.group;
            if (item.tiles > 0) {  // Q, swizzled as TMA would, a warp some of its rows; the products that read the last item's are done
                const T* q = static_cast<const T*>(p.a.q) + item.sequence * p.a.q_strides[0] + token * p.a.q_strides[1] +
                             query_head * p.a.q_strides[2];
                uint4 v[D / 8 / kGroups];
                by_rows<D, kGroups>(row <= last_row ? q : nullptr, group, [&](int i, int at_row, int c, const uint8_t* at) {
                    v[i] = at != nullptr ? reinterpret_cast<const uint4*>(at)[c] : make_uint4(0, 0, 0, 0);
                    // A BF16 row may not fit a half: see attend_kernel. Its D / 8 lanes have a piece each.
                    if constexpr (kCodes) row_scale[quarter * 32 + at_row] = to_halves<T, D / 8>(&v[i]);
                });
                by_rows<D, kGroups>(nullptr, group, [&](int i, int at, int c, const uint8_t*) { *tile_piece(queries, quarter * 32 + at, c) = v[i]; });
                fence_proxy_async();
                mbar_arrive(&q_full);
            }
            {
                uint32_t zero[32] = {};
#pragma unroll
                for (int c = 0; c < D / 32; ++c) tmem_store_32(tmem_o + c * 32, zero);
                tmem_store_wait();
            }
            const float base_scale = p.a.scale * kLog2e * (kCodes ? p.a.cache.k_scale[item.head] : 1.f);
            const float value_scale = kCodes ? p.a.cache.v_scale[item.head] : 1.f;
            float m = -INFINITY, l = 0.f;
            uint32_t own_steps = 0;  // of this group in this item
            for (int tile = 0; tile < item.tiles; ++tile, ++step) {
                if (step % kGroups != static_cast<uint32_t>(group)) {
                    if (++stage == kSteps) stage = 0;
                    continue;
                }
                const uint32_t s_at = tmem_s + mine + buffer(step) * 64, last_own = step - kGroups;
                uint32_t raw[64];
                wait(&s_full[buffer(step)], phase(step), 11, tile);
                tmem_load_32(s_at, raw);
                tmem_load_32(s_at + 32, raw + 32);
                tmem_load_wait();
                float (&s)[64] = reinterpret_cast<float(&)[64]>(raw);
                const int key0 = item.start + tile * kTileKeys;
                const uint64_t present = step_present[stage];
                const float scale = kCodes ? base_scale * row_scale[r] : base_scale;  // written before the scores were computed
                const bool by_row = key0 < all_from || key0 + kTileKeys > all_to;  // rows see different keys of this step
                const bool edge = by_row || present != ~0ull;
#pragma unroll
                for (int j = 0; j < 64; ++j) s[j] *= scale;
                if (edge) {
                    const int lo = from - key0, hi = to - key0;
#pragma unroll
                    for (int j = 0; j < 64; ++j)
                        if (j < lo || j >= hi || !(present >> j & 1)) s[j] = -INFINITY;
                }
                float top4[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                for (int j = 4; j < 64; ++j) top4[j & 3] = fmaxf(top4[j & 3], s[j]);
                const float top = fmaxf(fmaxf(top4[0], top4[1]), fmaxf(top4[2], top4[3]));
                if (__any_sync(0xFFFFFFFFu, top > m + (kRescaleAbove + kHeadroom<M>) || (m == -INFINITY && top > m))) {
                    const float n = fmaxf(m, top - kHeadroom<M>);
                    const float f = m == n ? 1.f : exp2_approx(m - n);  // 0 where nothing was there
                    l *= f, m = n;
                    if (own_steps > 0) {
                        wait(&pv_done[buffer(last_own)], phase(last_own), 12, tile);
#pragma unroll 1
                        for (int c = 0; c < D / 32; ++c) {
                            uint32_t o[32];
                            tmem_load_32(tmem_o + c * 32, o);
                            tmem_load_wait();
#pragma unroll
                            for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
                            tmem_store_32(tmem_o + c * 32, o);
                        }
                    }
                }
                const float sub = m == -INFINITY ? 0.f : m;
                float sum4[4] = {0.f, 0.f, 0.f, 0.f};
                uint32_t high[32], low[32];
#pragma unroll
                for (int j = 0; j < 64; j += 2) {
                    s[j] = exp2_approx(s[j] - sub), s[j + 1] = exp2_approx(s[j + 1] - sub);
                    sum4[j & 3] += s[j], sum4[(j + 1) & 3] += s[j + 1];
                    split_weights<M, kCodes>(s[j], s[j + 1], &high[j / 2], &low[j / 2]);
                }
                l += (sum4[0] + sum4[1]) + (sum4[2] + sum4[3]);
                tmem_store_32(s_at, high);
                tmem_store_32(s_at + 32, low);
                if (edge) {
                    // Values that are not finite, in keys that some rows see and others do not, or that are not there: 0 * inf
                    // would reach the result. Where there are any, every warp finds their keys for itself.
                    uint8_t* values = smem + stage * 2 * kBytes + kBytes;
                    auto piece = [&](int key, int c) {  // 16 bytes of a key's row
                        return reinterpret_cast<uint4*>(values + (c / 8) * kBlockBytes + key * 128 + ((c % 8) ^ (key & 7)) * 16);
                    };
                    uint32_t odd = 0;  // a quarter of the keys each warp, loads in flight together: 32 in a row took a microsecond
#pragma unroll
                    for (int i = 0; i < D / 16; ++i) {
                        const int at = i * 32 + lane;
                        const uint4 v = *piece(quarter * 16 + at / (D / 8), at % (D / 8));
                        odd |= not_finite<M>(v.x) | not_finite<M>(v.y) | not_finite<M>(v.z) | not_finite<M>(v.w);
                    }
                    uint64_t bad = 0;
                    if (group_any(group, odd != 0)) {
#pragma unroll 1
                        for (int i = 0; i < 2; ++i) {
                            const int key = lane + 32 * i;
                            bool any = false;
                            if (by_row || !(present >> key & 1)) {
                                for (int c = 0; c < D / 8; ++c) {
                                    const uint4 v = *piece(key, c);
                                    any |= (not_finite<M>(v.x) | not_finite<M>(v.y) | not_finite<M>(v.z) | not_finite<M>(v.w)) != 0;
                                }
                            }
                            bad |= static_cast<uint64_t>(__ballot_sync(0xFFFFFFFFu, any)) << (32 * i);
                        }
                    }
                    if (bad != 0) {  // the same in all warps of the group
                        uint64_t weightless = 0;  // keys whose weight is zero here: 0 * inf is NaN
#pragma unroll
                        for (int j = 0; j < 64; ++j) weightless |= static_cast<uint64_t>(s[j] == 0.f) << j;
                        if (own_steps > 0) wait(&pv_done[buffer(last_own)], phase(last_own), 13, tile);
                        tmem_store_wait();  // O may just have been rescaled
#pragma unroll 1
                        for (uint64_t left = bad; left != 0; left &= left - 1) {
                            const int key = __ffsll(static_cast<long long>(left)) - 1;
                            const bool see = key0 + key >= from && key0 + key < to && (present >> key & 1);
#pragma unroll 1
                            for (int c = 0; c < D / 32; ++c) {
                                uint32_t o[32];
                                tmem_load_32(tmem_o + c * 32, o);
                                tmem_load_wait();
#pragma unroll
                                for (int j = 0; j < 32; j += 2) {
                                    const uint32_t w = reinterpret_cast<const uint32_t*>(piece(key, c * 4 + j / 8))[j / 2 % 4];
                                    const float2 v = widen2<M>(w);
                                    const float none = weightless >> key & 1 ? NAN : 1.f;
                                    if (see && !isfinite(v.x)) o[j] = __float_as_uint(__uint_as_float(o[j]) + v.x * none);
                                    if (see && !isfinite(v.y)) o[j + 1] = __float_as_uint(__uint_as_float(o[j + 1]) + v.y * none);
                                }
                                tmem_store_32(tmem_o + c * 32, o);
                            }
                            tmem_store_wait();
                        }
                        mbar_arrive(&aside[group]);  // everybody has read them
                        wait(&aside[group], aside_parity, 14, tile);
                        aside_parity ^= 1;
                        for (uint64_t left = bad; left != 0; left &= left - 1) {
                            const int key = __ffsll(static_cast<long long>(left)) - 1;
                            if ((key & 3) != quarter) continue;
                            for (int c = lane; c < D / 8; c += 32) {
                                uint4 v = *piece(key, c);
                                v.x &= ~not_finite<M>(v.x), v.y &= ~not_finite<M>(v.y), v.z &= ~not_finite<M>(v.z), v.w &= ~not_finite<M>(v.w);
                                *piece(key, c) = v;
                            }
                        }
                        fence_proxy_async();
                    }
                }
                tmem_store_wait();
                tcgen05_fence_before();
                mbar_arrive(&p_full[buffer(step)]);
                ++own_steps;
                if (++stage == kSteps) stage = 0;
            }
            // -- the row's result ---------------------------------------------------------------------------------------
            if (own_steps > 0) {
                const uint32_t last_own = step - 1 - ((step - 1) % kGroups == static_cast<uint32_t>(group) ? 0 : 1);
                wait(&pv_done[buffer(last_own)], phase(last_own), 15, item.tiles);
            }
            // The groups' results together: every group takes its share of the elements, from each group's O.
            group_stats[group][r] = make_float2(m, l);
            rows_sync<kGroups>(quarter);
            float factors[kGroups];
            m = -INFINITY, l = 0.f;
#pragma unroll
            for (int i = 0; i < kGroups; ++i) m = fmaxf(m, group_stats[i][r].x);
#pragma unroll
            for (int i = 0; i < kGroups; ++i) {
                const float2 stats = group_stats[i][r];
                factors[i] = stats.x == -INFINITY ? 0.f : exp2_approx(stats.x - m);
                l += stats.y * factors[i];
            }
            // Parts of a row go out with rows side by side, [element / 4][row], a finished row by way of the tile of queries, whose
            // products are done: a thread's own row would be 32 lanes' stores far apart (5 us an item instead of 1.5).
            if (row <= last_row && group == 0) {
                if (!item.whole)
                    *reinterpret_cast<float2*>(p.stats + (static_cast<size_t>(item.piece) * p.rows_cap + r) * 2) = make_float2(m, l);
                else if (p.a.lse != nullptr)
                    p.a.lse[(static_cast<size_t>(item.sequence) * p.a.tokens + token) * p.a.q_heads + query_head] =
                        l == 0.f ? -INFINITY : (m + log2f(l)) * (1.f / kLog2e);
            }
            if (item.whole) {
                const float inv = l == 0.f ? 0.f : value_scale / l;
#pragma unroll
                for (int i = 0; i < kGroups; ++i) factors[i] *= inv;
            }
            constexpr int kChunks = D / 32 / kGroups;
#pragma unroll 1
            for (int c = group * kChunks; c < (group + 1) * kChunks; ++c) {
                float v[32];
#pragma unroll
                for (int i = 0; i < kGroups; ++i) {
                    uint32_t o[32];
                    tmem_load_32(tmem + mine + i * D + c * 32, o);
                    tmem_load_wait();
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] = (i == 0 ? 0.f : v[j]) + __uint_as_float(o[j]) * factors[i];
                }
                if (item.whole) {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        *tile_piece(queries, r, c * 4 + j) = make_uint4(narrow2<T>(v[8 * j], v[8 * j + 1]), narrow2<T>(v[8 * j + 2], v[8 * j + 3]),
                                                                        narrow2<T>(v[8 * j + 4], v[8 * j + 5]), narrow2<T>(v[8 * j + 6], v[8 * j + 7]));
                } else if (row <= last_row) {
                    float4* out = reinterpret_cast<float4*>(p.partial) + static_cast<size_t>(item.piece) * p.rows_cap * (D / 4) + r;
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        out[static_cast<size_t>(c * 8 + j) * p.rows_cap] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
                }
                __syncwarp();
            }
            if (item.whole) {
                rows_sync<kGroups>(quarter);
                __syncwarp();
                T* out = static_cast<T*>(p.a.out) + item.sequence * p.a.out_strides[0] + token * p.a.out_strides[1] +
                         query_head * p.a.out_strides[2];
                by_rows<D, kGroups>(row <= last_row ? out : nullptr, group, [&](int, int at, int c, uint8_t* to) {
                    if (to != nullptr) reinterpret_cast<uint4*>(to)[c] = *tile_piece(queries, quarter * 32 + at, c);
                });
                __syncwarp();
            }
            rows_sync<kGroups>(quarter);  // the next item's queries, statistics and O take the place of these
        }
    }
    tcgen05_fence_before();
    __syncthreads();
    if (warp == Shape::kIssuerWarp) {
        tcgen05_fence_after();
        tmem_dealloc(tmem, Shape::kColumns);
    }
}

// Joins the partial results of an item that lies in several runs (see SplitItem): 32 rows a block, a row each lane, the elements
// of a row shared among the warps. Finished rows go out by way of shared memory.
constexpr int kJoinRows = 32, kJoinWarps = 8;

template <typename T, int D>
__global__ void __launch_bounds__(kJoinWarps * 32) join_blocks_kernel(const __grid_constant__ AttendDev p) {
    constexpr int kMine = D / 4 / kJoinWarps;             // float4s of a row that a thread has
    constexpr int kAhead = D == 64 ? 8 : D == 128 ? 4 : 2;  // partial results on the way at once
    __shared__ __align__(16) uint8_t rows[kJoinRows][D * 2 + 16];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const SplitItem item(p, blockIdx.x);
    const int r = blockIdx.y * kJoinRows + lane, row = item.row_tile * kBlockRows + r;
    const bool there = r < p.rows_cap && row < p.rows;
    // Every block waits, those without work too: this kernel's end stands for the end of the one in front.
    pdl_wait();
    pdl_launch_dependents();
    if (!item.split) return;
    float4 sum[kMine];
#pragma unroll
    for (int i = 0; i < kMine; ++i) sum[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    float top = -INFINITY, l = 0.f;
    if (there) {
        for (int c0 = item.run; c0 <= item.last; c0 += kAhead) {
            float2 ml[kAhead];
            float4 v[kAhead][kMine];
#pragma unroll
            for (int a = 0; a < kAhead; ++a) {
                const int c = c0 + a;
                ml[a] = make_float2(-INFINITY, 0.f);
#pragma unroll
                for (int i = 0; i < kMine; ++i) v[a][i] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (c > item.last) continue;
                const size_t piece = static_cast<size_t>(c * 2 + (c == item.run));
                ml[a] = __ldcg(reinterpret_cast<const float2*>(p.stats) + piece * p.rows_cap + r);
#pragma unroll
                for (int i = 0; i < kMine; ++i)
                    v[a][i] = __ldcg(reinterpret_cast<const float4*>(p.partial) + (piece * (D / 4) + warp + i * kJoinWarps) * p.rows_cap + r);
            }
            float n = top;
#pragma unroll
            for (int a = 0; a < kAhead; ++a) n = fmaxf(n, ml[a].x);
            const float keep = top == -INFINITY ? 0.f : exp2_approx(top - n);
            l *= keep, top = n;
#pragma unroll
            for (int i = 0; i < kMine; ++i) sum[i].x *= keep, sum[i].y *= keep, sum[i].z *= keep, sum[i].w *= keep;
#pragma unroll
            for (int a = 0; a < kAhead; ++a) {
                const float f = ml[a].x == -INFINITY ? 0.f : exp2_approx(ml[a].x - n);
                l += ml[a].y * f;
#pragma unroll
                for (int i = 0; i < kMine; ++i)
                    sum[i].x += v[a][i].x * f, sum[i].y += v[a][i].y * f, sum[i].z += v[a][i].z * f, sum[i].w += v[a][i].w * f;
            }
        }
    }
    const float inv = l == 0.f ? 0.f : (p.a.cache.type == DLM_E4M3 ? p.a.cache.v_scale[item.head] : 1.f) / l;
    const int token = token_of(p, min(row, p.rows - 1)), query_head = item.head * p.group + min(row, p.rows - 1) - token * p.group;
#pragma unroll
    for (int i = 0; i < kMine; ++i)
        *reinterpret_cast<uint2*>(&rows[lane][(warp + i * kJoinWarps) * 8]) =
            make_uint2(narrow2<T>(sum[i].x * inv, sum[i].y * inv), narrow2<T>(sum[i].z * inv, sum[i].w * inv));
    if (there && warp == 0 && p.a.lse != nullptr)
        p.a.lse[(static_cast<size_t>(item.sequence) * p.a.tokens + token) * p.a.q_heads + query_head] =
            l == 0.f ? -INFINITY : (top + log2f(l)) * (1.f / kLog2e);
    __syncthreads();
    T* out = static_cast<T*>(p.a.out) + item.sequence * p.a.out_strides[0] + token * p.a.out_strides[1] + query_head * p.a.out_strides[2];
    by_rows<D, kJoinWarps>(there ? out : nullptr, warp, [&](int, int at, int c, uint8_t* to) {
        if (to != nullptr) reinterpret_cast<uint4*>(to)[c] = *reinterpret_cast<const uint4*>(&rows[at][c * 16]);
    });
}

int launch_blocks(const AttendDev& p, const LaunchOpts& o) {
    void* args[] = {const_cast<AttendDev*>(&p)};
    auto run = [&](auto t, auto dim, auto codes) {
        using T = decltype(t);
        constexpr int kDim = decltype(dim)::value;
        constexpr bool kCodes = decltype(codes)::value;
        using Shape = BlockShape<kDim, kCodes>;
        const int rc = launch_kernel<blocks_kernel<T, kDim, kCodes>>(dim3(p.grid), dim3(Shape::kThreads), Shape::kAll, args, o);
        if (rc != 0 || p.partial == nullptr) return rc;
        return launch_kernel<join_blocks_kernel<T, kDim>>(dim3(p.by_item ? p.a.batch * p.items : p.grid, (p.rows_cap + kJoinRows - 1) / kJoinRows),
                                                          dim3(kJoinWarps * 32), 0, args, {o.stream, true, false});
    };
    auto by_dim = [&](auto t, auto codes) {
        switch (p.a.cache.head_dim) {
            case 64: return run(t, std::integral_constant<int, 64>{}, codes);
            case 128: return run(t, std::integral_constant<int, 128>{}, codes);
            default: return run(t, std::integral_constant<int, 256>{}, codes);
        }
    };
    auto by_codes = [&](auto t) { return p.a.cache.type == DLM_E4M3 ? by_dim(t, std::true_type{}) : by_dim(t, std::false_type{}); };
    return p.a.type == DLM_F16 ? by_codes(__half{}) : by_codes(__nv_bfloat16{});
}

}  // namespace dlm
