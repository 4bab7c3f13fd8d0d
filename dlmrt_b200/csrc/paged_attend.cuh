// What both attention kernels over the paged cache share (paged_attend.cu, paged_blocks.cu): how the work is dealt out, the
// producer that requests keys and values, and how a row is finished.
//
// An item is one sequence, key head and row tile. The keys of all items are lined up in units of 64 keys and cut evenly into
// runs, one for each CTA that the GPU holds, whatever the lengths of the sequences. Requests go on across the items of a run. An
// item that lies in several runs leaves a partial result in each, which join_kernel adds up in their order. (SMs do not read
// equally fast, up to 30 % apart. Further, shorter runs, taken over by CTAs that get done early, cost more partial results and
// begun items than they gain: 64 ragged sequences 88.7 us with five waves of runs, 88.0 with two, 87.4 with one; 131071 keys 53.1 /
// 49.8 / 48.7; 64 sequences of 16 rows 45.1 / 38.8 / 35.4; FP8 heads of 256 84.8 / 80.0 / 80.2.)
//
// An item's beginning and end take time, too: its units begin with `lead` units without keys that stand for it. A run that
// holds only such units of an item leaves it to the next one.
#pragma once

#include <climits>

#include "mma.cuh"
#include "serving.cuh"

namespace dlm {

constexpr int kWorkSlots = 4;  // items that may be announced ahead
constexpr float kLog2e = 1.4426950408889634f;

// Weights are exp2(s - m) for a reference m that follows the running maximum: it is set to the maximum less kHeadroom, and anew
// when a score is more than kRescaleAbove past that. Weights then lie below 2^8, those that are taken as halves below 2^15. Halves
// end at 2^-24: with the largest weight at 2^7 the many small ones of a long cache keep 7 bits more (with m the maximum itself, keys
// 2^26 times lighter than the heaviest counted for nothing, and half of what 8000 of them add was lost). BF16 has the range of FP32.
constexpr float kRescaleAbove = 8.f;
template <typename M>
constexpr float kHeadroom = std::is_same<M, __half>::value ? 7.f : 0.f;
static_assert(kRescaleAbove + kHeadroom<__half> <= 15.f, "weights fit halves");

// Two weights as the product with the values takes them, which knows 16-bit types only: each as a high and a low part, whose
// products are added in FP32. One value alone is off by up to 2^-8 of the weight (BF16; halves 2^-11), which is more than the rounding
// of a result in which values partly cancel; both parts together are off by 2^-15 (halves: 2^-20, and 2^-25 of 1).
//
// Values of a 16-bit cache may be infinite. Neither part may then make a NaN of infinity, by its sign or by being zero: the high
// part is rounded towards zero, and less than the weight by 2^-12 of it and a step of halves at least; for BF16 2^-20 of the
// weight is added to the low part instead. FP8 has no infinity.
//
// What the second product costs: nothing where HBM bounds a call (64 ragged sequences 87.5 us with one part and with two, 131071
// keys 48.2 / 48.4, FP8 heads of 256 77.8 / 78.6), more where 16 rows share FP8 keys (heads of 256 78.5 / 86.0, of 128 33.6 / 35.9) and
// in blocks of tokens (16 of 32 tokens 58.7 / 63.0 us, call after call 64.9 / 73.1, most of it the product's tensor cycles; a prompt
// of 2048 tokens 108 / 118).
template <typename M, bool kCodes>
__device__ __forceinline__ void split_weights(float x, float y, uint32_t* high, uint32_t* low) {
    if constexpr (!std::is_same<M, __half>::value) {
        constexpr float kMore = 1.f + 0x1p-20f;
        const uint32_t a = __float_as_uint(x), b = __float_as_uint(y);
        *high = __byte_perm(a, b, 0x7632);
        *low = narrow2<M>(fmaf(x, kMore, -__uint_as_float(a & 0xFFFF0000u)), fmaf(y, kMore, -__uint_as_float(b & 0xFFFF0000u)));
    } else {
        if constexpr (kCodes) {
            *high = narrow2<M>(x, y);
        } else {
            constexpr float kLess = 1.f - 0x1p-12f, kStep = -0x1p-24f;
            *high = narrow2_down_to_zero(fmaf(x, kLess, kStep), fmaf(y, kLess, kStep));
        }
        const float2 h = widen2<M>(*high);
        *low = narrow2<M>(x - h.x, y - h.y);
    }
}

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
    s.base = (p.a.window > 0 ? max(0, s.first_pos - p.a.window + 1) : 0) & ~(kTileKeys - 1);
    s.units = p.lead + max(1, static_cast<int>((static_cast<uint32_t>(s.length - s.base) + (1u << p.unit_shift) - 1) >> p.unit_shift));
    return s;
}
// Keys that a token sees: [seen_from, seen_to).
__device__ __forceinline__ int seen_from(const AttendDev& p, int first_pos, int token) {
    return p.a.window > 0 ? max(0, first_pos + token - p.a.window + 1) : 0;
}
__device__ __forceinline__ int seen_to(const AttendDev& p, int first_pos, int length, int token) {
    return p.a.causal ? min(length, first_pos + token + 1) : length;
}

// The token that a row (query head of the group, token) belongs to.
__device__ __forceinline__ int token_of(const AttendDev& p, int row) { return p.a.tokens == 1 ? 0 : row / p.group; }

// The line of units and its runs. Every warp that needs it works it out for itself: a lane looks at a range
// of the sequences. The host has seen to it that there are fewer than 2^31 units.
struct Line {
    uint32_t total;
    int runs;
    int first, last;    // this lane's sequences
    uint32_t before;    // units in front of them
    uint32_t mine;      // units of them

    __device__ __forceinline__ Line(const AttendDev& p, bool tell) {
        const int lane = threadIdx.x & 31;
        const int per = (p.a.batch + 31) >> 5;
        first = min(lane * per, p.a.batch), last = min(first + per, p.a.batch);
        mine = 0;
        for (int i = first; i < last; ++i) mine += sequence_of(p, i, tell).units;
        mine *= p.items;
        before = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t up = __shfl_up_sync(0xFFFFFFFFu, before, o);
            if (lane >= o) before += up;
        }
        total = __shfl_sync(0xFFFFFFFFu, before, 31);
        before -= mine;
        runs = attend_runs(total, p.resident);
    }
    // The units [begin, end) of a run: dealt out evenly, rounded down, and no run is empty.
    __device__ __forceinline__ void range(int run, uint32_t* begin, uint32_t* end) const {
        const uint32_t across = runs, i = run, each = total / across, over = total - each * across;
        *begin = each * i + over * i / across;
        *end = each * (i + 1) + over * (i + 1) / across;
    }
    __device__ __forceinline__ int run_of(uint32_t unit) const {
        return static_cast<int>((static_cast<unsigned long long>(unit + 1) * runs - 1) / total);
    }
    // The units in front of a sequence. All lanes of the warp.
    __device__ __forceinline__ uint32_t in_front_of(const AttendDev& p, int sequence) const {
        const int per = (p.a.batch + 31) >> 5, holder = sequence / per;
        uint32_t front = __shfl_sync(0xFFFFFFFFu, before, holder);
        for (int i = holder * per; i < sequence; ++i) front += static_cast<uint32_t>(sequence_of(p, i, false).units) * p.items;
        return front;
    }
    // The sequence that holds a unit, and the units in front of that sequence. All lanes of the warp.
    __device__ __forceinline__ int sequence_at(const AttendDev& p, uint32_t unit, uint32_t* in_front) const {
        int sequence = first;
        uint32_t front = before;
        const bool here = unit >= before && unit < before + mine;
        if (here) {
            for (; sequence < last - 1; ++sequence) {
                const uint32_t units = static_cast<uint32_t>(sequence_of(p, sequence, false).units) * p.items;
                if (unit < front + units) break;
                front += units;
            }
        }
        const uint32_t holder = __ballot_sync(0xFFFFFFFFu, here);
        const int from = holder ? __ffs(holder) - 1 : 0;
        *in_front = __shfl_sync(0xFFFFFFFFu, front, from);
        return __shfl_sync(0xFFFFFFFFu, sequence, from);
    }
};

// What those who compute have to know of an item in a run.
struct Work {
    int sequence, head, row_tile;  // head -1: there is no more work
    int length, first_pos;
    int start, end, tiles;         // keys of this run, steps of 64 of them
    int whole;                     // all keys of the item are in this run
    int piece;                     // otherwise: index of its partial result
};

// The rings between the producer and the warps that compute: stages of keys and values, and announced items.
template <int kStages>
struct alignas(16) Pipes {
    uint64_t full[kStages], empty[kStages], present[kStages];  // present: bit j says that the stage's key j is there
    uint64_t work_full[kWorkSlots], work_empty[kWorkSlots];
    Work works[kWorkSlots];

    // One thread; `readers` arrive for every stage that they are done with, `listeners` for every item.
    __device__ __forceinline__ void init(int readers, int listeners) {
        for (int i = 0; i < kStages; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], readers);
        for (int i = 0; i < kWorkSlots; ++i) mbar_init(&work_full[i], 1), mbar_init(&work_empty[i], listeners);
        fence_barrier_init();
    }
};

// Until when a role waits that begins an item now: a call of many items may take longer than a wait that nothing will end.
__device__ __forceinline__ long long item_deadline() { return globaltimer() + kDefaultTimeoutNs; }

// How long a block whose waits ran out waits for what it has on the way itself.
constexpr long long kDrainNs = 1000000000ll;

// A wait that runs out is reported; what follows is computed from whatever is there, and nothing more is requested.
__device__ __forceinline__ void stalled(const AttendDev& p, int who, int at) {
    report(p.a.cache.status, kErrTimeout, who, kPhasePipeline, at);
}

// The producer: a whole warp. A stage of the ring is kPieces * 16 bytes for each of 64 keys, then the same for values. Boxes
// are a page's slots, at most 64; kApart: of one column block of 128 bytes each, so that a block's 64 rows follow one another.
template <int kStages, int kPieces, bool kApart>
__device__ __forceinline__ void produce(const AttendDev& p, uint8_t* ring, Pipes<kStages>& pipes, bool leader) {
    const int lane = threadIdx.x & 31;
    constexpr int kBytes = kTileKeys * kPieces * 16;
    constexpr int kBlocks = kApart ? (kPieces + 7) / 8 : 1;  // boxes along a row
    const Line line(p, blockIdx.x == 0);
    const int box_keys = min(kTileKeys, 1 << p.page_shift), boxes = kTileKeys / box_keys;
    const int slot_mask = (1 << p.page_shift) - 1;
    const int run = blockIdx.x;
    int stage = 0, slot = 0;
    uint32_t parity = 1, slot_parity = 1;  // the first lap of a ring waits for nothing
    bool failed = false;
    long long deadline = item_deadline();
    auto announce = [&](const Work& work) {
        if (!mbar_wait_warp(&pipes.work_empty[slot], slot_parity, deadline) && !failed) {
            failed = true;
            if (leader) stalled(p, 0, run);
        }
        if (leader) {
            pipes.works[slot] = work;
            mbar_arrive(&pipes.work_full[slot]);
        }
        if (++slot == kWorkSlots) slot = 0, slot_parity ^= 1;
    };
    // Where the next step is: an item in the run, a step of 64 keys in that. Pages are looked up a step ahead of their use,
    // across items, 32 entries of the table at once: lane j holds entry `window` + j.
    uint32_t unit = 0, last_unit = 0;
    int sequence = 0, index = 0, first = 0, units = 0, lo = 0, tile = 0, window = 0, pages = 0;
    Sequence s{};
    Work work{};
    auto look_up = [&](int from) {
        window = from;
        const int entry = from + lane;
        pages = entry << p.page_shift < work.end ? p.a.page_table[sequence * p.a.table_stride + entry] : INT_MIN;
    };
    auto begin_item = [&]() {
        units = min(static_cast<int>(last_unit - unit), s.units - first);
        work.sequence = sequence, work.length = s.length, work.first_pos = s.first_pos;
        work.head = p.row_tiles == 1 ? index : index / p.row_tiles, work.row_tile = index - work.head * p.row_tiles;
        const int first_row = work.row_tile * p.tile_rows, last_row = min(first_row + p.tile_rows, p.rows) - 1;
        lo = seen_from(p, s.first_pos, token_of(p, first_row));
        const int hi = seen_to(p, s.first_pos, s.length, token_of(p, last_row));
        const int end = first + units - p.lead, begin = max(0, first - p.lead);  // in units with keys
        work.whole = first <= p.lead && first + units == s.units;
        work.piece = run * 2 + (first <= p.lead);  // a run has at most one that began before it and one that goes on
        work.start = max(s.base + (begin << p.unit_shift), lo & ~(kTileKeys - 1));  // begin is 0 if units are whole items
        work.end = first + units == s.units ? hi : min(hi, s.base + (max(0, end) << p.unit_shift));
        work.tiles = end <= 0 ? -1 : work.end > work.start ? (work.end - work.start + kTileKeys - 1) / kTileKeys : 0;
        tile = 0;
        deadline = item_deadline();
        if (work.tiles > 0) look_up(work.start >> p.page_shift);
    };
    auto begin_run = [&]() -> bool {
        if (run >= line.runs) return false;
        line.range(run, &unit, &last_unit);
        uint32_t in_front;
        sequence = line.sequence_at(p, unit, &in_front);
        s = sequence_of(p, sequence, false);
        index = static_cast<int>((unit - in_front) / static_cast<uint32_t>(s.units));  // key head * row tiles + row tile
        first = static_cast<int>(unit - in_front) - index * s.units;
        begin_item();
        return true;
    };
    auto advance = [&]() -> bool {
        if (++tile < work.tiles) {
            const int entry = (work.start + tile * kTileKeys) >> p.page_shift;
            if (entry >= window + 32) look_up(entry);
            return true;
        }
        unit += units;
        if (unit < last_unit) {
            first = 0;
            if (++index == p.items) index = 0, s = sequence_of(p, ++sequence, false);
            begin_item();
            return true;
        }
        return false;
    };
    bool more = begin_run();
    while (more) {
        const Work now = work;
        const int now_tile = tile, now_lo = lo;
        const int now_pages = pages, now_window = window;
        more = advance();
        if (now.tiles < 0) continue;  // the next run's
        if (now_tile == 0) announce(now);
        if (now.tiles == 0) continue;
        const int key0 = now.start + now_tile * kTileKeys;
        // Lane j: the page of box j, INT_MIN where no key of the box is in the run.
        const int entry = ((key0 + lane * box_keys) >> p.page_shift) - now_window;
        int page = __shfl_sync(0xFFFFFFFFu, now_pages, entry & 31);
        const bool in_pool = static_cast<uint32_t>(page) < static_cast<uint32_t>(p.a.cache.pages);
        uint64_t present = ~0ull;
        if (!__all_sync(0xFFFFFFFFu, in_pool || lane >= boxes) || now.end - key0 < kTileKeys) {
            if (lane >= boxes || key0 + lane * box_keys >= now.end) page = INT_MIN;
            else if (!in_pool && key0 + (lane + 1) * box_keys > now_lo)
                report_index(p.a.cache.status, now.sequence, kIndexPage, page);
            const uint32_t there = __ballot_sync(0xFFFFFFFFu, in_pool && page != INT_MIN);
            if (!in_pool || page == INT_MIN) page = p.a.cache.pages;  // past the pool's end: the box is filled with zeros
            const uint64_t box_bits = box_keys == 64 ? ~0ull : (1ull << box_keys) - 1;
            present = 0;
            for (int j = 0; j < boxes; ++j)
                if (there >> j & 1) present |= box_bits << (j * box_keys);
            if (now.end - key0 < kTileKeys) present &= (1ull << (now.end - key0)) - 1;
        }
        if (!mbar_wait(&pipes.empty[stage], parity, deadline) && !failed) {
            failed = true;
            if (leader) stalled(p, 1, now_tile);
        }
        __syncwarp();
        uint8_t* to = ring + stage * 2 * kBytes;
        uint64_t* bar = &pipes.full[stage];
        if (leader) {
            pipes.present[stage] = present;
            if (failed) mbar_arrive(bar);
            else mbar_expect_tx(bar, 2 * kBytes);
        }
        for (int j = 0; j < boxes; ++j) {
            const int from = __shfl_sync(0xFFFFFFFFu, page, j);
            const int at = (key0 + j * box_keys) & slot_mask;
            const int box = j * box_keys * (kApart && kPieces > 8 ? 128 : kPieces * 16);
            if (leader && !failed) {
#pragma unroll
                for (int c = 0; c < kBlocks; ++c) {
                    tma_load_5d(to + c * kTileKeys * 128 + box, &p.tm_k, bar, 0, at, c, now.head, from, kEvictNormal);
                    tma_load_5d(to + kBytes + c * kTileKeys * 128 + box, &p.tm_v, bar, 0, at, c, now.head, from, kEvictNormal);
                }
            }
        }
        if (++stage == kStages) stage = 0, parity ^= 1;
    }
    if (failed) {
        // Copies that are still on the way would otherwise land in memory that another block has by then. `stage` is the next one to
        // be filled: those in front of it were filled in this lap, the others in the one before.
        const long long limit = globaltimer() + kDrainNs;
        for (int i = 0; i < kStages; ++i) mbar_wait(&pipes.full[i], i < stage ? parity ^ 1 : parity, limit);
    }
    Work none;
    none.head = -1;
    announce(none);
}

// What a block of a join looks at: an item that lies in several runs. Block `b` has item b, or (with more items than runs) the
// item that begins in run b and goes on. All threads; lengths are older than the kernel in front, whose blocks waited for them
// before a dependent launch could start, so this need not wait.
struct SplitItem {
    bool split;
    int sequence, head, row_tile, run, last;  // its runs are [run, last]

    __device__ __forceinline__ SplitItem(const AttendDev& p, int b) : split(false), sequence(0), head(0), row_tile(0), run(b), last(b) {
        const Line line(p, false);
        int index;
        if (p.by_item) {
            sequence = b / p.items, index = b - sequence * p.items;
            const Sequence s = sequence_of(p, sequence, false);
            const uint32_t begin = line.in_front_of(p, sequence) + index * s.units;
            run = line.run_of(begin + p.lead), last = line.run_of(begin + s.units - 1);
            split = last != run;
        } else {
            run = b;
            if (run + 1 >= line.runs) return;
            uint32_t run_begin, run_end, in_front;
            line.range(run, &run_begin, &run_end);
            sequence = line.sequence_at(p, run_end - 1, &in_front);
            const Sequence s = sequence_of(p, sequence, false);
            index = static_cast<int>((run_end - 1 - in_front) / static_cast<uint32_t>(s.units));
            const uint32_t begin = in_front + index * s.units;
            last = line.run_of(begin + s.units - 1);
            split = begin + p.lead >= run_begin && begin + p.lead < run_end && last != run;
        }
        head = index / p.row_tiles, row_tile = index - head * p.row_tiles;
    }
};

// Four elements of a finished row: the sum over its keys, divided by the sum of their weights.
template <typename T>
__device__ __forceinline__ void finish_row(const AttendDev& p, int sequence, int head, int row, int d, const float4& sum,
                                           float top, float l, float value_scale) {
    const float inv = l == 0.f ? 0.f : value_scale / l;
    const int token = token_of(p, row), query_head = head * p.group + row - token * p.group;
    T* out = static_cast<T*>(p.a.out) + sequence * p.a.out_strides[0] + token * p.a.out_strides[1] +
             query_head * p.a.out_strides[2] + d;
    *reinterpret_cast<uint2*>(out) = make_uint2(narrow2<T>(sum.x * inv, sum.y * inv), narrow2<T>(sum.z * inv, sum.w * inv));
    if (p.a.lse != nullptr && d == 0)
        p.a.lse[(static_cast<size_t>(sequence) * p.a.tokens + token) * p.a.q_heads + query_head] =
            l == 0.f ? -INFINITY : (top + log2f(l)) * (1.f / kLog2e);
}

}  // namespace dlm
