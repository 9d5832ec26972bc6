// Operators of the layers between leaf vectors and classes: the root-mean-square
// norm and its gradient, rows to 8 bits and back, projections with adapters and
// their gradients. Called as the operators over leaves (leafops.h) are.
#pragma once
#include <cstdint>

#include "hessboost_rocm.h"

namespace hbr {

void rms_norm(int ordinal, void *stream, const hbr_norm &p);
uint64_t rms_norm_grad_workspace(uint64_t n_rows, uint32_t dim, uint32_t dtype);
void rms_norm_grad(int ordinal, void *stream, const hbr_norm_grad &p, void *workspace, uint64_t workspace_bytes);

void pack_rows(int ordinal, void *stream, const hbr_packed &p, const void *x, uint8_t *codes, uint8_t *scales);
void unpack_rows(int ordinal, void *stream, const hbr_packed &p, const uint8_t *codes, const uint8_t *scales,
                 const float *weight, void *x);

uint64_t linear_workspace(uint64_t n_rows, uint32_t outs, uint32_t dim, uint32_t rank, uint32_t dtype);
void linear(int ordinal, void *stream, const hbr_linear_args &p, void *workspace, uint64_t workspace_bytes);
uint64_t linear_grad_workspace(uint64_t n_rows, uint32_t outs, uint32_t dim, uint32_t dtype);
void linear_grad(int ordinal, void *stream, const hbr_linear_grad_args &p, void *workspace, uint64_t workspace_bytes);

}  // namespace hbr
