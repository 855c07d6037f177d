// How the 64-key tiles of sparse attention's units, (kv head, tile of prompt rows)
// pairs one after another, are dealt to workgroups in equal runs, and where the parts of
// units that a run's end cuts leave their partials.  Plain arithmetic, which the plan and
// the kernel share.
#pragma once
#include <stdint.h>

#ifdef __HIP__
#define GLLM_RUNS __host__ __device__ inline
#else
#define GLLM_RUNS inline
#endif

namespace gllm {

// Blocks whose ids, rows and numbers a workgroup holds for a run: a run of whole 64-key tiles
// may start and end inside blocks, so one block less of keys and one to spare.
constexpr int kRunCache = 1024;
GLLM_RUNS int64_t most_run_tiles(int32_t block_size) { return (int64_t)(kRunCache - 2) * block_size / 64; }
// Runs of C >= 1 tiles: `round` at a time (one a CU), in as many rounds as that takes, but of
// four tiles at least.  Grows with C.
GLLM_RUNS int64_t tile_runs(int64_t C, int64_t round, int32_t block_size) {
  const int64_t a_round = round * most_run_tiles(block_size);
  const int64_t full = (C + a_round - 1) / a_round * round, short_ones = C / 4 > 1 ? C / 4 : 1;
  return short_ones < full ? short_ones : full;
}
// Run r has the tiles [run_start(r), run_start(r + 1)); run_of(s) is the one with tile s.
GLLM_RUNS int64_t run_start(int64_t C, int64_t runs, int64_t r) { return C * r / runs; }
GLLM_RUNS int64_t run_of(int64_t C, int64_t runs, int64_t s) { return ((s + 1) * runs - 1) / C; }

// The run of a workgroup (past the last run: none).  Workgroups go to the 8 XCDs in turn:
// neighbouring runs, which share keys, on one XCD, and every XCD has its share of the runs
// that there are, however many the plan launches workgroups for.
GLLM_RUNS int64_t run_of_group(int64_t group, int64_t runs) {
  return group < runs && runs % 8 == 0 ? group % 8 * (runs / 8) + group / 8 : group;
}

// Slots of partials.  Only a run's first and last unit can be parts: two slots a run, of
// which the first unit takes the even one; where there are fewer units than runs one a run
// and one a unit are less.
GLLM_RUNS int64_t run_slots(int64_t runs, int64_t units) { return runs + (units < runs ? units : runs); }
GLLM_RUNS int32_t part_slot(int64_t runs, int64_t units, int64_t run, int64_t unit, bool first_of_run) {
  return (int32_t)(units < runs ? run + unit : 2 * run + (first_of_run ? 0 : 1));
}
// The partials of a unit: slot first, then rest, rest + step, ... (count in all; 1: none, the
// output is written).
struct TileParts {
  int32_t first, rest, step, count;
};
// Of unit `unit`, which has the c tiles from s0 on.
GLLM_RUNS TileParts unit_parts(int64_t C, int64_t runs, int64_t units, int64_t unit, int64_t s0, int64_t c) {
  const int64_t r0 = run_of(C, runs, s0), r1 = run_of(C, runs, s0 + c - 1);
  return {part_slot(runs, units, r0, unit, run_start(C, runs, r0) >= s0), part_slot(runs, units, r0 + 1, unit, true),
          units < runs ? 1 : 2, (int32_t)(r1 - r0 + 1)};
}

}  // namespace gllm
