// mx_columns.hpp -- which rows of w a group of the few-rows product reads, and which columns of
// the output it holds.  Plain functions, compiled for the device by the kernel and for the host by a test.
#pragma once

#ifdef __HIPCC__
#define NPU_MX_HD __host__ __device__ __forceinline__
#else
#define NPU_MX_HD inline
#endif

namespace npu {

// Group i of 16 nt columns, from n0 on; each column is one group's, so that the last group may
// have less (or tiles without any).
struct FewColumns {
  long long n0;
  int last;  // the last row of w, from n0
  NPU_MX_HD FewColumns(int i, int nt, int N) : n0((long long)i * (16 * nt)), last((int)(N - 1 - n0)) {}
  // The row, from n0, that row r of a tile reads: past the last one the last again.
  NPU_MX_HD int row(int tile, int r) const { return 16 * tile + r < last ? 16 * tile + r : last; }
  // The first of the four columns that lane group g holds of a tile: a multiple of 4, on which the
  // workspace's vectors lie.  None of the four is stored where it is N or more.
  NPU_MX_HD long long first(int tile, int g) const { return n0 + 16 * tile + 4 * g; }
};

}  // namespace npu
