// block_norm.cuh - norms before and after a block (block_norm.cu): what the C ABI hands to the launchers.
#pragma once

#include "moe_internal.cuh"

struct NormCall {
  pm_norm_desc D;  // strides filled in
  int T;
  float inv_d;     // 1 / d
  bool vec;        // every row of every stream and every weight starts on 16 bytes, rows are whole 16-byte words
  const void *x, *f, *w_post, *gate, *w_pre;  // x: of the gradient, the stream behind the block
  // forward
  void *r, *n;
  // gradient
  const void *dr, *dn;
  void *dx, *df;
  float *dw_post, *dgate, *dw_pre;
  float *parts;    // norm_parts_floats(D, T, n_sm) floats
};

size_t norm_parts_floats(const pm_norm_desc &D, int T, int n_sm);
cudaError_t launch_block_norm(const Launch &L, const NormCall &c);
cudaError_t launch_block_norm_grad(const Launch &L, const NormCall &c);
