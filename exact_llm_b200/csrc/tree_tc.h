// Tree attention on tcgen05 (tree_tc.cu), used by exb_tree_attention.
#pragma once
#include "treedev.cuh"

namespace exb {

struct TtWork {
  unsigned long long* rowmax = nullptr;      // (R, H) maxima in unsigned order, 0: nothing seen
  unsigned long long* rowsum = nullptr;      // (R, H) sums of e
  int64_t* pre = nullptr;                    // 2 x (B + 1): units before each sequence, by row tiles of the two kinds
};
size_t tt_workspace_bytes(int R, int H, int B);
cudaError_t launch_tree_tc(const TreeArgs& a, void* workspace, cudaStream_t st);

}  // namespace exb
