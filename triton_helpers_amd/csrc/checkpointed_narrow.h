// The linear layer with 8-bit checkpoints for many rows and at most 256 channels on either side: the layer's weights stay with a workgroup, and a row
// is read and written once in the forward and once in the backward (checkpointed_narrow.hip).
#pragma once

#include "nf_common.h"

namespace nf {

struct NarrowFwd {
  const void *x, *w, *bias;
  void* y;
  int8_t* q;  // NULL: nothing is kept
  float* scale;
  int64_t xs, ws, ys, rows;
  int n, k, bias_dt, act;
};
struct NarrowBwd {
  const void *dy, *w;  // w, dx: NULL where no dx is wanted
  const int8_t* q;
  const float* scale;
  void* dx;
  float *dw, *db;  // [groups][n][k], [groups][n]: partial sums of each workgroup (db: NULL where it is not wanted)
  int64_t dys, ws, rows;
  int n, k, act;
};

// Whether these kernels take the call: rows and weights on 16-byte boundaries, whole 16-byte pieces, enough rows to share the weights.
bool narrow_fits(int64_t rows, int64_t n, int64_t k);
int narrow_groups(int64_t rows);  // workgroups of the backward
int narrow_fwd(const NarrowFwd& a, int dtype, hipStream_t s);
int narrow_bwd(const NarrowBwd& a, int dtype, hipStream_t s);

}  // namespace nf
