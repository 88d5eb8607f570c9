// Where a cut of the attention's line of work falls in a unit.  Plain C++, so
// that it can be compiled and looked at without a GPU.
#pragma once

#ifdef __CUDACC__
#define SVD_LINE_FN __host__ __device__ __forceinline__
#else
#define SVD_LINE_FN inline
#endif

namespace svdmlp {

// A unit takes `cost` places of the line for itself and then one for each of
// its `steps`.  The step before which a cut `in` places behind its beginning
// (0 <= in < cost + steps) divides it: 0 the unit's start, `steps` the next
// one's.  A unit of at most `snap` steps is not divided, its cuts go to the nearer
// end.  In a longer one the cuts within its cost go to its start: were the last of
// them sent to the next unit, a cut behind them would lie before them, and its
// steps would be done twice.
SVD_LINE_FN int cut_step(int in, int steps, int cost, int snap) {
  if (steps <= snap) return 2 * in > steps + cost ? steps : 0;
  return in > cost ? in - cost : 0;
}

}  // namespace svdmlp
