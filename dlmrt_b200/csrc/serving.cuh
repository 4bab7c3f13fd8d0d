// What the paged cache's and the adapters' kernels share with the C boundary: parameter blocks, launchers, and how an
// index that lies outside its table is reported.
#pragma once

#include "../../include/dlmrt_b200.h"
#include "kernels.cuh"

namespace dlm {

// Which index was out of range: the `slot` of the status words (their `block` is the row or sequence, `epoch` the value; of a slot
// of the cache `epoch` is its page and `phase` the place in it).
enum IndexKind { kIndexSlot = 1, kIndexPosition = 2, kIndexPage = 3, kIndexLength = 4, kIndexAdapter = 5 };

// First error wins, as report(). The words describe a row instead of a block.
__device__ __forceinline__ void report_index(int* status, int row, int kind, int value, int place = 0) {
    if (status == nullptr) return;
    if (atomicCAS(status, 0, DLM_ERR_INDEX) == 0) {
        status[1] = (row << 8) | kind;
        status[2] = place;
        status[3] = value;
    }
}

constexpr int kFewRows = 8, kRowTile = 16;  // rows of an item: the N of its matrix instructions, once or twice
constexpr int kBlockRows = 128;  // the same in the kernel for blocks of tokens
constexpr int kUnitShift = 6, kTileKeys = 1 << kUnitShift;  // keys of a step, and of the units that items are cut into

struct alignas(64) AttendDev {
    CUtensorMap tm_k, tm_v;  // (128 bytes, page size, column blocks, heads, pages); a box: min(page size, kTileKeys) whole slots
    DlmAttend a;
    float* partial;    // [run][2][rows_cap][head_dim] unnormalised outputs of items that lie in several runs, or null; in the
                       // kernel for blocks of tokens [run][2][head_dim / 4][rows_cap][4]
    float* stats;      // the same without head_dim, 2: running maximum (base 2) and sum
    int page_shift;
    int group;         // query heads of a key head
    int rows;          // tokens * group rows share a key head's keys
    int tile_rows;     // rows of an item: kFewRows, kRowTile, or kBlockRows in the kernel for blocks of tokens
    int row_tiles;     // of tile_rows rows
    int rows_cap;      // rows of a tile that exist: min(tile_rows, rows)
    int blocks;        // the kernel for blocks of tokens takes this call
    int items;         // of one sequence: key heads * row tiles
    int unit_shift;    // log2 of the keys of a unit: kUnitShift, or more than there are where items are not split
    int lead;          // units that an item has in front of those with keys: what its beginning and end cost
    int resident;      // CTAs that the GPU holds
    int grid;          // CTAs, and runs that there are at most
    int by_item;       // the join has a block for each item, not for each run
    int sms;
};

// How many runs a line of `total` units is cut into: one for each CTA that the GPU holds, or for each unit of a short line.
__host__ __device__ inline int attend_runs(uint32_t total, int resident) {
    return total < static_cast<uint32_t>(resident) ? static_cast<int>(total) : resident;
}

int launch_append(const DlmAppend& p, int page_shift, const LaunchOpts& o);
int launch_attend(const AttendDev& p, const LaunchOpts& o);
int launch_blocks(const AttendDev& p, const LaunchOpts& o);
int attend_ctas_per_sm(int type, int cache_type, int head_dim, int tile_rows);
int launch_adapters(const DlmAdapters& p, const LaunchOpts& o);

}  // namespace dlm
