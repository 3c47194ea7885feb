// adapter.h -- low-rank adapters of a projection's rows (internal to the
// library).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace llm {

constexpr uint32_t kAdapterRankMax = 512;

// The rows of one adapter (a null: rows without any, rank 0).
struct AdapterGroup {
    const int16_t* a;  // [rank][inputs] Q4.12
    const int16_t* b;  // [rank][outputs] Q4.12
    uint32_t rank;
    int32_t scale;     // Q16.16
    uint32_t rows;     // how many, and which
    uint8_t row[8];
};
struct AdapterArgs {
    AdapterGroup g[8];
    uint32_t groups;
    uint32_t ranks;       // of all groups together
    uint32_t start[8];    // ranks of the groups before each (no group: ~0)
    const int16_t* x;     // rows [][inputs], tight
    uint32_t inputs, outputs;
    int32_t* t;           // [8][kAdapterRankMax] Q16.16: x A^T
    const int64_t* wide;  // the projection's exact sums [][outputs], 20 fraction bits
    int16_t* out;         // rows [][outputs], tight
};
// t = sat32(rnd(x A^T, 4)) of every row with an adapter: by workgroups of the
// projection's own launch (EPI_WIDE, adapter_in.h).
// out = narrow(wide + rnd(scale sat32(rnd(t B, 12)), 12)).
hipError_t launch_adapter_out(const AdapterArgs& a, hipStream_t st);

}  // namespace llm
