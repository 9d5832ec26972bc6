// Operators over leaves and many classes: leaf vectors looked up and their
// table's gradient, the softmax head, gradient clipping. Each queues its
// kernels on the caller's stream and keeps what it needs meanwhile in the
// caller's workspace: nothing is allocated, copied or waited for, so a call
// can be captured into a graph. Arguments are checked before the device is touched.
#pragma once
#include <cstdint>

#include "hessboost_rocm.h"
#include "runtime.h"

namespace hbr {

void leaf_embedding(int ordinal, void *stream, const hbr_lookup &p, const void *table, void *out);
uint64_t leaf_embedding_grad_workspace(const hbr_lookup &p);
void leaf_embedding_grad(int ordinal, void *stream, const hbr_lookup &p, const void *dout, void *dtable,
                         void *workspace, uint64_t workspace_bytes);

uint64_t softmax_head_workspace(uint64_t n_rows, uint32_t n_classes, uint32_t dim, uint32_t dtype, bool gradient);
void softmax_head(int ordinal, void *stream, const hbr_softmax &p, void *workspace, uint64_t workspace_bytes);

uint64_t clip_gradients_workspace(uint64_t n_tensors);
void clip_gradients(int ordinal, void *stream, const hbr_tensor *tensors, uint64_t n, double max_norm, float *norm,
                    void *workspace, uint64_t workspace_bytes);

}  // namespace hbr
