// tree_tile.cuh -- host interface of the tensor-memory variant of the draft-tree attention.
#pragma once

#include "tree_common.cuh"

namespace ckl {
namespace tree {

// Row tiles of 128 that a CTA holds for up to `rows` stacked rows.
int tile_count(long long rows);
// Bytes of partials of `ctas` CTAs.
size_t tile_workspace(int ctas, long long rows);
// Checked parameters and filled arguments (out, lse set) -> both kernels on `s`.
ckl_status launch_tiles(const ckl_tree_params* p, Args a, void* workspace, int ctas, cudaStream_t s);

}  // namespace tree
}  // namespace ckl
