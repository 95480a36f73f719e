// 8-bit rows, activations that keep them, and edge attention (torch_rows8.cpp).
#pragma once
#include "torch_ops.h"

namespace tango_host {

// An 8-bit copy of a tensor seen as a matrix [size(0), rest] (1-D: one row): codes [rows, ld] int8, scales [rows, groups] fp32.
struct Rows8 {
    Tensor q, scale;
};
Rows8 pack8(const Tensor &x, int64_t group);
// The values as a new tensor of `sizes` and `type`. `like` (one element at least) tells its type.
Tensor unpack8(const Rows8 &r, at::IntArrayRef sizes, int64_t group, at::ScalarType type);

// f(x), the backward pass from an 8-bit copy of x; act: 0 ELU, 1 GELU (erf), 2 SiLU.
Tensor activation8_fn(const Tensor &x, int act, int64_t group);

// Dot-product attention of every node over its incoming edges, q, k, v [N, H, D] held in 8 bits with a scale per node and head.
Tensor edge_attention_fn(const GraphPtr &g, const Tensor &q, const Tensor &k, const Tensor &v, double scale);
// The same for the nodes `rows` only, with their queries [R, H, D], over packed keys and values; no gradient.
Tensor edge_attention_rows(const GraphPtr &g, const Tensor &rows, const Tensor &q, const Rows8 &k, const Rows8 &v, double scale);

}  // namespace tango_host
