// tree_tile.cuh -- host interface of the tensor-memory variant of the draft-tree attention.
#pragma once

#include "tree_common.cuh"

namespace ckl {
namespace tree {

// K or V cache as pages of one head, a box of [halves][16 tokens][64 dims].
ckl_status encode_half_map(const void* cache, int Hkv, int num_pages, int halves, CUtensorMap* tm);
// q [N][Hq][128] as boxes of [tokens][heads][64 dims]: stacked rows in order.
ckl_status encode_q_map(const void* q, int N, int Hq, int heads, int tokens, CUtensorMap* tm);
// Row tiles of 128 that a CTA holds for up to `rows` stacked rows.
int tile_count(long long rows);
// Bytes of partials of `ctas` CTAs.
size_t tile_workspace(int ctas, long long rows);
// Checked parameters and filled arguments (out, lse set) -> both kernels on `s`.
ckl_status launch_tiles(const ckl_tree_params* p, Args a, void* workspace, int ctas, cudaStream_t s);

}  // namespace tree
}  // namespace ckl
