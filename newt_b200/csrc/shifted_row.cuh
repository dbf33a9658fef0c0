// Where the columns of a row lie that is read in vectors from its first vector boundary on.  Plain
// arithmetic, so that it can be looked at without a GPU.
#pragma once

#ifndef __CUDACC__
#define __host__
#define __device__
#define __forceinline__ inline
#endif

namespace nb200 {

// A row of n columns that starts m elements behind a boundary of E-element vectors: columns
// [head, end) are whole vectors, the others are taken one by one.  A thread's vectors start at
// columns `lane * E - m` and multiples of the row's step further; the first of them begins in front of
// the row where m is not 0 and is left out.  Groups are 2^group_shift >= E columns, counted from column 0,
// so a vector's first m columns are in one group and the others in one group.
struct ShiftedRow {
  int n, m, head, end;

  __host__ __device__ __forceinline__ ShiftedRow(int n, int m, int E) : n(n), m(m), head(m ? E - m : 0) {
    const int inner = n - m - head;      // a vector of the weight's second half ends inside the row too
    end = head + (inner > 0 ? inner : 0) / E * E;
  }
  // is there a vector at this column?
  __host__ __device__ __forceinline__ bool whole(int column) const { return (unsigned)column < (unsigned)end; }
  // how many columns are taken one by one, and the i-th of them
  __host__ __device__ __forceinline__ int singles() const { return n - (end - head); }
  __host__ __device__ __forceinline__ int single(int i) const { return i < head ? i : end - head + i; }
  // the group of the first m columns of the vector at `column`, -1: there are none
  __host__ __device__ __forceinline__ int group_before(int column, int group_shift) const {
    return m && whole(column) ? (column + m - 1) >> group_shift : -1;
  }
  // the group of E neighbours from a multiple of E on: the others of the vector at `column` and the
  // first m of the next one; -1: behind the row
  __host__ __device__ __forceinline__ int group_from(int column, int group_shift) const {
    return column + m < n ? (column + m) >> group_shift : -1;
  }
};

}  // namespace nb200
