// What the paged cache's and the adapters' kernels share with the C boundary: parameter blocks, launchers, and how an
// index that lies outside its table is reported.
#pragma once

#include "../../include/dlmrt_b200.h"
#include "kernels.cuh"

namespace dlm {

// Which index was out of range: the `slot` of the status words (their `block` is the row or sequence, `epoch` the value).
enum IndexKind { kIndexSlot = 1, kIndexPosition = 2, kIndexPage = 3, kIndexLength = 4, kIndexAdapter = 5 };

// First error wins, as report(). The words describe a row instead of a block.
__device__ __forceinline__ void report_index(int* status, int row, int kind, int value) {
    if (status == nullptr) return;
    if (atomicCAS(status, 0, DLM_ERR_INDEX) == 0) {
        status[1] = (row << 8) | kind;
        status[2] = 0;
        status[3] = value;
    }
}

constexpr int kRowTile = 16;   // rows of an item: the M of its matrix instructions
constexpr int kUnitKeys = 64;  // keys of the smallest piece of work that items are cut into

struct AttendDev {
    DlmAttend a;
    float* partial;    // [cta][2][rows_cap][head_dim] unnormalised outputs of items that lie in several CTAs' runs, or null
    float* stats;      // the same without head_dim, 2: running maximum (base 2) and sum
    int page_shift;
    int group;         // query heads of a key head
    int rows;          // tokens * group rows share a key head's keys
    int row_tiles;     // of kRowTile rows
    int rows_cap;      // rows of a tile that exist: min(kRowTile, rows)
    int items;         // of one sequence: key heads * row tiles
    int unit;          // keys of a unit; the table's length where items are not split
    int least_units;   // of a run
    int ctas;
};

int launch_append(const DlmAppend& p, int page_shift, const LaunchOpts& o);
int launch_attend(const AttendDev& p, const LaunchOpts& o);
int attend_ctas_per_sm(int type, int cache_type, int head_dim);
int launch_adapters(const DlmAdapters& p, const LaunchOpts& o);

}  // namespace dlm
