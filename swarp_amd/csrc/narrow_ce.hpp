// narrow_ce.hpp -- linear_ce.hip and narrow_ce.hip, of each other.
#pragma once
#include "learn.hpp"

namespace narrow {

constexpr int COUNT_ROWS = 4096;  // rows of a mask that one number stands for

inline int64_t counts_of(int64_t rows) { return (rows + COUNT_ROWS - 1) / COUNT_ROWS; }
// linear_ce.hip: how many rows count, of every COUNT_ROWS.
void count(int64_t rows, const uint8_t *mask, int32_t *counts, hipStream_t st);

// narrow_ce.hip: whether a head's weight fits a workgroup's LDS, the work memory of a call, and the
// call: gradients (NULL: not wanted) for the upstream gradient *scale (NULL: 1; with skip_unit they
// are there already where it is 1).
bool fits(const swarp_linear_ce_t *a);
uint64_t work_bytes(const swarp_linear_ce_t *a);
int run(const swarp_linear_ce_t *a, int skip_unit, const float *scale, void *d_hidden, void *d_weight, void *d_bias,
        hipStream_t st);

}  // namespace narrow
