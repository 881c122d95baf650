// The products and the cache operators of torch_binding.cpp as functions: what the operators of their names
// do on CUDA tensors, with all their checks. torch_direct.cpp calls them without the operator dispatcher.
#pragma once

#include <ATen/core/Tensor.h>

#include <cstdint>
#include <optional>

namespace macko_torch {

// y[rows] for V[cols]. `flags`: MACKO_SPMV_MATRIX_IMMUTABLE, MACKO_SPMV_ROWS_EVEN.
at::Tensor multiply_flags(const at::Tensor &values, const at::Tensor &deltas, const at::Tensor &ri, int64_t rows, int64_t cols,
                          const at::Tensor &V, uint32_t flags);

at::Tensor multiply_planned_cuda(const at::Tensor &values, const at::Tensor &deltas, const at::Tensor &ri, int64_t rows, int64_t cols,
                                 const at::Tensor &plan, int64_t virtual_rows, int64_t segment_elements, int64_t split_rows,
                                 const at::Tensor &V, bool frozen);

// y[batch, rows] for V[batch, cols] over the matrix's column windows.
at::Tensor multiply_windowed_cuda(const at::Tensor &values, const at::Tensor &deltas, const at::Tensor &ri, int64_t rows, int64_t cols,
                                  const at::Tensor &windows, const at::Tensor &V, bool frozen);

// Dense [rows, cols] of a compressed matrix.
at::Tensor decompress_cuda(const at::Tensor &values, const at::Tensor &deltas, const at::Tensor &ri, int64_t rows, int64_t cols);

// q [rows, heads, head_dim], rotated, for qkv [rows, (heads + 2 kv_heads) head_dim]; k and v go into the cache.
at::Tensor rope_append_cuda(const at::Tensor &qkv, const at::Tensor &cos_table, const at::Tensor &sin_table, at::Tensor k_cache,
                            at::Tensor v_cache, at::Tensor k_scale, at::Tensor v_scale, const at::Tensor &page_table,
                            const at::Tensor &lengths, const std::optional<at::Tensor> &query_start);

// Attention of q [rows, heads, head_dim] over the cache.
at::Tensor paged_attention_cuda(const at::Tensor &q, const at::Tensor &k_cache, const at::Tensor &v_cache, const at::Tensor &k_scale,
                                const at::Tensor &v_scale, const at::Tensor &page_table, const at::Tensor &lengths,
                                const std::optional<at::Tensor> &query_start, std::optional<double> scale);

}  // namespace macko_torch
