// fna2_paged_books.h — the books of a paged cache on the GPU: launches.
#pragma once

#include "fna2_paged.h"

namespace fna2 {

struct BooksParams {
  int N, width, ps, cap;  // sequences, entries of a table row, rows of a page, entries of the stack
  uint32_t ps_mul;        // as in PagedParams
  int ps_shift;
  int64_t tstride;
  int* table;
  const int* lens;
  const int* counts;  // extend: new tokens; trim: rows to keep
  int* free;          // stack of free pages, the first *nfree of them in use
  const int* nfree;
  int* new_lens;
  int* new_nfree;
  // extend
  int T;
  const int* shift;  // [N], or null
  int* cu;           // [N + 1]
  int64_t* slots;    // [T]
  int* seq;          // [T]
  int* pos;          // [T]
  int* status;       // [1]
  // trim
  const int* borrowed;  // [N], or null
  // groups
  int* common;      // [N] workspace
  int* cu_groups;   // [N + 1]
  int* shared_rows; // [N]
};

hipError_t launch_paged_extend(const BooksParams& P, hipStream_t s);
hipError_t launch_paged_trim(const BooksParams& P, hipStream_t s);
hipError_t launch_paged_groups(const BooksParams& P, hipStream_t s);

}  // namespace fna2
