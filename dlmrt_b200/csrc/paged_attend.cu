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
// Each of a CTA's four warps takes every fourth tile of 16 keys through a ring of its own (cp.async, no block-wide step in
// the main loop), with its own maximum, sum and output in registers; the four are joined in shared memory.
//
// Work is dealt out evenly, whatever the lengths: the keys of all items (an item: one sequence, key head and row tile) are
// lined up in units of 64, and each of as many CTAs as the GPU holds at once takes one contiguous run of units. It goes
// through the items of its run without draining the ring in between, so one item's end overlaps the next one's loads. An
// item that lies in several runs leaves a partial result in each, which join_kernel adds up in order. Every CTA reads all
// lengths and works its run out by itself.
#include "mma.cuh"
#include "serving.cuh"

namespace dlm {

namespace {

constexpr int kAttendWarps = 4;
constexpr int kAttendThreads = kAttendWarps * 32;
constexpr int kTileKeys = 16;
constexpr int kJoinRows = 4;  // rows of a tile that the warps exchange at a time
constexpr float kLog2e = 1.4426950408889634f;

// A sequence's keys: how many, the position of its first new token, where its units begin, and how many an item of it has.
struct Sequence {
    int length, first_pos, base, units;
};

__device__ __forceinline__ Sequence sequence_of(const AttendDev& p, int index, bool tell) {
    Sequence s;
    const long long room = static_cast<long long>(p.a.table_pages) << p.page_shift;
    const int length = p.a.lengths[index];
    s.length = length < 0 ? 0 : length > room ? static_cast<int>(room) : length;
    if (tell && s.length != length) report_index(p.a.cache.status, index, kIndexLength, length);
    s.first_pos = s.length - p.a.tokens;
    s.base = (p.a.window > 0 ? max(0, s.first_pos - p.a.window + 1) : 0) & ~(kUnitKeys - 1);
    s.units = max(1, (s.length - s.base + p.unit - 1) / p.unit);
    return s;
}
// Keys that a token sees: [seen_from, seen_to).
__device__ __forceinline__ int seen_from(const AttendDev& p, const Sequence& s, int token) {
    return p.a.window > 0 ? max(0, s.first_pos + token - p.a.window + 1) : 0;
}
__device__ __forceinline__ int seen_to(const AttendDev& p, const Sequence& s, int token) {
    return p.a.causal ? min(s.length, s.first_pos + token + 1) : s.length;
}

// The line of units: `total` of them over `ctas` CTAs, the first `extra` of which have one more than `each`.
struct Line {
    long long total, each;
    int ctas, extra;
    __device__ long long begin(int cta) const { return each * cta + min(cta, extra); }
    __device__ int owner(long long unit) const {
        const long long longer = (each + 1) * extra;
        return static_cast<int>(unit < longer ? unit / (each + 1) : extra + (unit - longer) / each);
    }
};

struct Place {  // of a unit: its sequence, and the units in front of that sequence
    int sequence;
    long long before;
};

// Works out the line, and where unit `of(line)` lies. All threads of the block (a multiple of 32, at most 256).
template <int kThreads, typename F>
__device__ __forceinline__ Line lay_out(const AttendDev& p, int ctas, bool tell, F of, long long* unit, Place* place) {
    __shared__ long long warp_sum[kThreads / 32];
    __shared__ Place found;
    const int tid = threadIdx.x, lane = tid & 31;
    const int per = (p.a.batch + kThreads - 1) / kThreads;
    const int first = min(tid * per, p.a.batch), last = min(first + per, p.a.batch);
    long long mine = 0;
    for (int i = first; i < last; ++i) mine += static_cast<long long>(sequence_of(p, i, tell).units) * p.items;
    long long before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xFFFFFFFFu, before, o);
        if (lane >= o) before += up;
    }
    if (lane == 31) warp_sum[tid >> 5] = before;
    before -= mine;
    if (tid == 0) found.sequence = p.a.batch, found.before = 0;
    __syncthreads();
    Line line;
    line.total = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
        if (w == tid >> 5) before += line.total;
        line.total += warp_sum[w];
    }
    const long long most = (line.total + p.least_units - 1) / p.least_units;
    line.ctas = static_cast<int>(most < ctas ? most : ctas);
    line.each = line.total / line.ctas;
    line.extra = static_cast<int>(line.total % line.ctas);
    *unit = of(line);
    if (*unit >= before && *unit < before + mine) {
        for (int i = first; i < last; ++i) {
            const long long units = static_cast<long long>(sequence_of(p, i, false).units) * p.items;
            if (*unit < before + units) {
                found.sequence = i, found.before = before;
                break;
            }
            before += units;
        }
    }
    __syncthreads();
    *place = found;
    return line;
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

constexpr int kStages = 3;

// Dynamic shared memory: the warps' rings, four rows of each warp's output, and (kQueriesInShared) the A operands of all
// k16 steps, in the order of the lanes.
template <int D, bool kCodes>
struct AttendSmem {
    static constexpr bool kQueriesInShared = D == 256;  // 64 registers of queries and 128 of output leave too few
    static constexpr int kRing = kStages * kAttendWarps * 2 * Stage<D, kCodes>::kBytes;
    static constexpr int kPitch = D + 4;
    static constexpr int kJoin = kAttendWarps * kJoinRows * kPitch * 4;
    static constexpr int kQueries = kQueriesInShared ? D / 16 * 512 : 0;
    static constexpr int kBytes = kRing + kJoin + kQueries;
    // CTAs that an SM holds; registers are held to what they leave each other.
    static constexpr int kCtas = D == 256 ? (kCodes ? 2 : 1) : D == 128 ? (kCodes ? 3 : 2) : 4;
};

}  // namespace

// Four elements of a finished row: the sum over its keys, divided by the sum of their weights.
template <typename T>
__device__ __forceinline__ void finish_row(const AttendDev& p, int sequence, int head, int row, int d, const float4& sum,
                                           float top, float l, float value_scale) {
    const float inv = l == 0.f ? 0.f : value_scale / l;
    const int token = row / p.group, query_head = head * p.group + row - token * p.group;
    T* out = static_cast<T*>(p.a.out) + sequence * p.a.out_strides[0] + token * p.a.out_strides[1] +
             query_head * p.a.out_strides[2] + d;
    *reinterpret_cast<uint2*>(out) = make_uint2(narrow2<T>(sum.x * inv, sum.y * inv), narrow2<T>(sum.z * inv, sum.w * inv));
    if (p.a.lse != nullptr && d == 0)
        p.a.lse[(static_cast<size_t>(sequence) * p.a.tokens + token) * p.a.q_heads + query_head] =
            l == 0.f ? -INFINITY : (top + log2f(l)) * (1.f / kLog2e);
}

// T: type of queries and output. Products are of T, or of halves where the cache holds FP8 codes (every code is a half).
template <typename T, int D, bool kCodes>
__global__ void __launch_bounds__(kAttendThreads, AttendSmem<D, kCodes>::kCtas) attend_kernel(const __grid_constant__ AttendDev p) {
    using M = typename std::conditional<kCodes, __half, T>::type;
    using S = Stage<D, kCodes>;
    using Shared = AttendSmem<D, kCodes>;
    constexpr int kSteps = D / 16;       // k16 steps of q . k
    constexpr int kOut = D / 8;          // n8 tiles of the output
    constexpr int kElem = kCodes ? 1 : 2;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float warp_stats[kAttendWarps][kRowTile][2];
    __shared__ uint32_t present_keys[kAttendWarps][4];
    __shared__ float weights_of_tile[kAttendWarps][kRowTile][kTileKeys + 1];

    const int warp = uniform(static_cast<int>(threadIdx.x >> 5)), lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const int cta = blockIdx.x;
    pdl_wait();
    pdl_launch_dependents();
    long long unit;
    Place place;
    const Line line = lay_out<kAttendThreads>(p, gridDim.x, cta == 0, [&](const Line& l) { return l.begin(cta); }, &unit, &place);
    if (cta >= line.ctas) return;
    const long long last_unit = line.begin(cta + 1);

    // Where an item of this run is, and which of its keys are in it.
    struct Item {
        Sequence s;
        int sequence, index;     // index: key head * row tiles + row tile
        int head, row_tile;
        int first, units;        // units of this run
        int start, end;          // their keys, as far as some row of the tile sees them
        int tiles;               // of 16 keys
        int lo;                  // first key that some row sees
    };
    auto narrow_to_run = [&](Item& item, long long left) {
        item.head = item.index / p.row_tiles, item.row_tile = item.index - item.head * p.row_tiles;
        item.units = static_cast<int>(left < item.s.units - item.first ? left : item.s.units - item.first);
        const int first_row = item.row_tile * kRowTile, last_row = min(first_row + kRowTile, p.rows) - 1;
        item.lo = seen_from(p, item.s, first_row / p.group);
        const int hi = seen_to(p, item.s, last_row / p.group);
        const long long to = item.s.base + static_cast<long long>(item.first + item.units) * p.unit;
        item.start = max(item.s.base + item.first * p.unit, item.lo & ~(kTileKeys - 1));
        item.end = static_cast<int>(to < hi ? to : hi);
        item.tiles = item.end > item.start ? (item.end - item.start + kTileKeys - 1) / kTileKeys : 0;
    };
    auto next_item = [&](Item& item, long long left) {
        item.first = 0;
        if (++item.index == p.items) {
            item.index = 0;
            item.s = sequence_of(p, ++item.sequence, false);
        }
        narrow_to_run(item, left);
    };
    Item item;
    item.sequence = place.sequence;
    item.s = sequence_of(p, item.sequence, false);
    {
        const long long inside = unit - place.before;
        item.index = static_cast<int>(inside / item.s.units);
        item.first = static_cast<int>(inside - static_cast<long long>(item.index) * item.s.units);
    }
    narrow_to_run(item, last_unit - unit);

    // -- the ring: this warp's tiles of all items of the run, one after the other ----------------------------------------
    uint8_t* ring = smem + warp * (kStages * 2 * S::kBytes);
    const uint32_t ring_u32 = smem_u32(ring);
    const long long k_page = p.a.cache.k_strides[0] * kElem, k_slot = p.a.cache.k_strides[2] * kElem;
    const long long v_page = p.a.cache.v_strides[0] * kElem, v_slot = p.a.cache.v_strides[2] * kElem;
    const int slot_mask = (1 << p.page_shift) - 1;
    Item ahead = item;                       // the item whose tiles are being requested
    long long ahead_left = last_unit - unit; // units of the run from its beginning on
    int ahead_tile = warp;
    int page_ahead = -1;                     // lane r of the lower half: page of key r of the tile to be requested next
    auto settle = [&]() -> bool {            // moves `ahead` to an item that still has a tile for this warp; fetches its pages
        while (ahead_tile >= ahead.tiles) {
            ahead_left -= ahead.units;
            if (ahead_left <= 0) return false;
            next_item(ahead, ahead_left);
            ahead_tile = warp;
        }
        const int key = ahead.start + ahead_tile * kTileKeys + lane;
        page_ahead = -1;
        if (lane < kTileKeys && key < ahead.end) {
            const int page = p.a.page_table[ahead.sequence * p.a.table_stride + (key >> p.page_shift)];
            if (page >= 0 && page < p.a.cache.pages) page_ahead = page;
            else if (key >= ahead.lo) report_index(p.a.cache.status, ahead.sequence, kIndexPage, page);
        }
        return true;
    };
    bool more = settle();
    auto issue = [&](int stage) {
        if (more) {
            const int page = page_ahead;
            const uint32_t present = __ballot_sync(0xFFFFFFFFu, page >= 0);
            if (lane == 0) present_keys[warp][stage] = present;
            const int key0 = ahead.start + ahead_tile * kTileKeys;
            const uint8_t* keys = static_cast<const uint8_t*>(p.a.cache.keys) + ahead.head * p.a.cache.k_strides[1] * kElem;
            const uint8_t* values = static_cast<const uint8_t*>(p.a.cache.values) + ahead.head * p.a.cache.v_strides[1] * kElem;
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
            ahead_tile += kAttendWarps;
            more = settle();
        }
        cp_async_commit();
    };
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) issue(s);
    int stage = 0, fill = kStages - 1;

    while (true) {
    const int sequence = item.sequence, head = item.head, row_tile = item.row_tile;
    // This thread's two rows: g and g + 8 of the tile.
    const int row0 = row_tile * kRowTile + g, row1 = row0 + 8;
    const int token0 = min(row0, p.rows - 1) / p.group, token1 = min(row1, p.rows - 1) / p.group;
    const int from0 = seen_from(p, item.s, token0), to0 = seen_to(p, item.s, token0);
    const int from1 = seen_from(p, item.s, token1), to1 = seen_to(p, item.s, token1);
    const int last_row = min(row_tile * kRowTile + kRowTile, p.rows) - 1;
    const int all_from = seen_from(p, item.s, last_row / p.group);               // from here on every row sees the keys
    const int all_to = seen_to(p, item.s, (row_tile * kRowTile) / p.group);      // up to here

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

    const uint32_t* shared_q = nullptr;
    if constexpr (Shared::kQueriesInShared) {
        uint32_t* to = reinterpret_cast<uint32_t*>(smem + Shared::kRing + Shared::kJoin);
        if (warp == 0) {
#pragma unroll
            for (int s = 0; s < kSteps; ++s)
                *reinterpret_cast<uint4*>(to + (s * 32 + lane) * 4) = make_uint4(q[s][0], q[s][1], q[s][2], q[s][3]);
        }
        __syncthreads();
        shared_q = to + lane * 4;
    }

    float o[kOut][4];
#pragma unroll
    for (int i = 0; i < kOut; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;

    for (int tile = warp; tile < item.tiles; tile += kAttendWarps) {
        cp_async_wait<kStages - 2>();
        __syncwarp();  // every lane's copies of this stage have landed, and every lane is done with the stage before
        issue(fill);
        const int key0 = item.start + tile * kTileKeys;
        const uint8_t* stage_k = ring + stage * 2 * S::kBytes;
        const uint32_t stage_k32 = ring_u32 + stage * 2 * S::kBytes, stage_v32 = stage_k32 + S::kBytes;
        const uint32_t present = present_keys[warp][stage];

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
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                uint32_t a[4], b[4];
                query_step(k, a);
                ldmatrix_x4(b, stage_k32 + (r * S::kPieces + S::key_piece(r, 2 * k + ((lane >> 3) & 1))) * 16);
                mma_16816<M>(s[0], a, b[0], b[1]);
                mma_16816<M>(s[1], a, b[2], b[3]);
            }
        } else {
#pragma unroll
            for (int k4 = 0; k4 < kSteps / 4; ++k4) {
                uint32_t a[4][4];
#pragma unroll
                for (int j = 0; j < 4; ++j) query_step(4 * k4 + j, a[j]);
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const int r = g + 8 * n;
                    const uint4 w = *reinterpret_cast<const uint4*>(stage_k + (r * S::kPieces + S::key_piece(r, 4 * k4 + t)) * 16);
                    const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        mma_16816<M>(s[n], a[j], e4m3x2_to_f16x2(words[j] & 0xFFFFu), e4m3x2_to_f16x2(words[j] >> 16));
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

    // -- the four warps' results, four rows at a time ---------------------------------------------------------------
#pragma unroll
    for (int x = 1; x < 4; x <<= 1) {
        l0 += __shfl_xor_sync(0xFFFFFFFFu, l0, x);
        l1 += __shfl_xor_sync(0xFFFFFFFFu, l1, x);
    }
    if (t == 0) {
        warp_stats[warp][g][0] = m0, warp_stats[warp][g][1] = l0;
        warp_stats[warp][g + 8][0] = m1, warp_stats[warp][g + 8][1] = l1;
    }
    __syncthreads();
    {
        float n0 = -INFINITY, n1 = -INFINITY;
#pragma unroll
        for (int w = 0; w < kAttendWarps; ++w) n0 = fmaxf(n0, warp_stats[w][g][0]), n1 = fmaxf(n1, warp_stats[w][g + 8][0]);
        // A warp that met no visible key has all zeros, or NaN times zero from a score that was NaN: kept as it is.
        const float f0 = m0 == -INFINITY ? 0.f : exp2_approx(m0 - n0), f1 = m1 == -INFINITY ? 0.f : exp2_approx(m1 - n1);
#pragma unroll
        for (int i = 0; i < kOut; ++i) o[i][0] *= f0, o[i][1] *= f0, o[i][2] *= f1, o[i][3] *= f1;
    }
    const int rows = min(kRowTile, p.rows - row_tile * kRowTile);
    const bool whole = item.units == item.s.units;
    const float value_scale = kCodes ? p.a.cache.v_scale[head] : 1.f;
    float* joined = reinterpret_cast<float*>(smem + Shared::kRing);
    for (int r0 = 0; r0 < rows; r0 += kJoinRows) {
        if ((g & ~(kJoinRows - 1)) == (r0 & 7)) {
            float* to = joined + (warp * kJoinRows + (g & (kJoinRows - 1))) * Shared::kPitch;
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
        __syncthreads();
        for (int i = threadIdx.x; i < min(kJoinRows, rows - r0) * (D / 4); i += kAttendThreads) {
            const int r = r0 + i / (D / 4), d = (i % (D / 4)) * 4;
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
            float top = -INFINITY, l = 0.f;
#pragma unroll
            for (int w = 0; w < kAttendWarps; ++w) {
                const float4 v = *reinterpret_cast<const float4*>(joined + (w * kJoinRows + (r - r0)) * Shared::kPitch + d);
                sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
                top = fmaxf(top, warp_stats[w][r][0]);
            }
#pragma unroll
            for (int w = 0; w < kAttendWarps; ++w) {
                const float m = warp_stats[w][r][0];
                l += warp_stats[w][r][1] * (m == -INFINITY ? 0.f : exp2_approx(m - top));
            }
            if (whole) {
                finish_row<T>(p, sequence, head, row_tile * kRowTile + r, d, sum, top, l, value_scale);
            } else {  // a run has at most two partial results: of an item that began in front of it, and of one that goes on
                const int piece = (cta * 2 + (item.first == 0)) * p.rows_cap + r;
                *reinterpret_cast<float4*>(p.partial + static_cast<size_t>(piece) * D + d) = sum;
                if (d == 0) *reinterpret_cast<float2*>(p.stats + piece * 2) = make_float2(top, l);
            }
        }
        __syncthreads();
    }
    unit += item.units;
    if (unit >= last_unit) break;
    next_item(item, last_unit - unit);
    }
    cp_async_wait<0>();
}

// Joins the partial results of the item that begins in run blockIdx.x and goes on in later ones: for each of its rows,
// out = sum_c exp2(m_c - m) o_c / sum_c exp2(m_c - m) l_c. D / 4 threads cover a row, the others further partial results.
// gridDim.y blocks share the rows of an item.
constexpr int kJoinThreads = 256;

template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const __grid_constant__ AttendDev p) {
    constexpr int kAcross = D / 4, kDeep = kJoinThreads / kAcross;
    __shared__ float4 sums[kDeep][kAcross];
    __shared__ float ls[kDeep];
    const int cta = blockIdx.x;
    // The lengths are older than the kernel in front, whose blocks waited for them before this one could start.
    long long unit;
    Place place;
    const Line line = lay_out<kJoinThreads>(p, gridDim.x, false, [&](const Line& l) { return l.begin(min(cta, l.ctas - 1) + 1) - 1; },
                                            &unit, &place);
    if (cta + 1 >= line.ctas) return;
    const Sequence s = sequence_of(p, place.sequence, false);
    const int index = static_cast<int>((unit - place.before) / s.units);
    const long long begin = place.before + static_cast<long long>(index) * s.units;
    const int head = index / p.row_tiles, first_row = (index - head * p.row_tiles) * kRowTile;
    const int last = line.owner(begin + s.units - 1);
    if (begin < line.begin(cta) || last == cta) return;
    pdl_wait();
    pdl_launch_dependents();
    const int x = threadIdx.x % kAcross, y = threadIdx.x / kAcross;
    for (int r = blockIdx.y; r < p.rows_cap && first_row + r < p.rows; r += gridDim.y) {
        auto piece = [&](int c) { return (c * 2 + (c == cta)) * p.rows_cap + r; };
        float top = -INFINITY;
        for (int c = cta; c <= last; ++c) top = fmaxf(top, __ldcg(p.stats + piece(c) * 2));
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        float l = 0.f;
#pragma unroll 4
        for (int c = cta + y; c <= last; c += kDeep) {
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(p.stats + piece(c) * 2));
            const float4 v = __ldcg(reinterpret_cast<const float4*>(p.partial + static_cast<size_t>(piece(c)) * D + x * 4));
            const float f = ml.x == -INFINITY ? 0.f : exp2_approx(ml.x - top);
            l += ml.y * f;
            sum.x += v.x * f, sum.y += v.y * f, sum.z += v.z * f, sum.w += v.w * f;
        }
        sums[y][x] = sum;
        if (x == 0) ls[y] = l;
        __syncthreads();
        if (y == 0) {
#pragma unroll
            for (int i = 1; i < kDeep; ++i) {
                const float4 v = sums[i][x];
                sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
                l += ls[i];
            }
            finish_row<T>(p, place.sequence, head, first_row + r, x * 4, sum, top, l,
                          p.a.cache.type == DLM_E4M3 ? p.a.cache.v_scale[head] : 1.f);
        }
        __syncthreads();
    }
}

template <typename T, int D, bool kCodes>
static int launch_attend_t(const AttendDev& p, const LaunchOpts& o) {
    void* args[] = {const_cast<AttendDev*>(&p)};
    const int rc = launch_kernel<attend_kernel<T, D, kCodes>>(dim3(p.ctas), dim3(kAttendThreads), AttendSmem<D, kCodes>::kBytes,
                                                              args, o);
    if (rc != 0 || p.partial == nullptr) return rc;
    // Few items: many partial results each, a block for every row. Many items: one or two each, and a block has to find out
    // first whether there is anything to join (0.5 us, and 9000 blocks took 25).
    const bool few = static_cast<long long>(p.a.batch) * p.items * 4 <= p.ctas;
    return launch_kernel<join_kernel<T, D>>(dim3(p.ctas, few ? p.rows_cap : 1), dim3(kJoinThreads), 0, args,
                                            {o.stream, true, false});  // always a dependent launch of the kernel above
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
    return by_type(p.a.type, p.a.cache.type, p.a.cache.head_dim, [&](auto t, auto dim, auto codes) {
        return launch_attend_t<decltype(t), decltype(dim)::value, decltype(codes)::value>(p, o);
    });
}

int attend_ctas_per_sm(int type, int cache_type, int head_dim) {
    return by_type(type, cache_type, head_dim,
                   [&](auto, auto dim, auto codes) { return AttendSmem<decltype(dim)::value, decltype(codes)::value>::kCtas; });
}

}  // namespace dlm
