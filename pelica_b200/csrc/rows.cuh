// rows.cuh - tokens sorted by expert and back (rows.cu): what the C ABI hands to the launchers.
#pragma once

#include "moe_internal.cuh"

// pairs (tokens x top_k) whose sort every CTA of the copy makes for itself
#define PM_ROWS_SMALL_PAIRS 1024
// value of a context's device error word: a row position in a device buffer that the plan's rows do not have
#define PM_DEVERR_BAD_ROW 101

struct RowsCall {
  pm_rows_desc D;   // strides and n_local filled in
  pm_rows_plan pl;
  int T;
  bool vec;         // every row of every buffer starts on 16 bytes and is whole 16-byte words
  int *err;         // the context's error word
};

// the plan; where x is given, the rows too (w: null, or the weights that scale them)
cudaError_t launch_rows_dispatch(const Launch &L, const RowsCall &c, const uint32_t *ids, const float *w, bool scale, const void *x, void *rows);
// out[t] = add[t] + sum_k w rows[pos]; dw[t][k] = <rows[pos], x[t]> where dw is given
cudaError_t launch_rows_gather(const Launch &L, const RowsCall &c, const float *w, const void *rows, const void *add, const void *x, void *out,
                               float *dw);
// out[pos] = w src[t], zeros in the padding; dw[t][k] = <rows[pos], src[t]> where dw is given
cudaError_t launch_rows_spread(const Launch &L, const RowsCall &c, const float *w, const void *src, const void *rows, void *out, float *dw);
