// tree.cuh -- what the kernels of tree attention share (tree.cu, tree_tc.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace gncx {

struct TreeArgs {
    const float* q;
    const float* kc;
    const float* vc;
    const int32_t* parents;
    int pos0, n_tok, n_heads, n_kv, hd, G;
    float scale2;      // softmax scale * log2(e): scores are exponents of 2
    int window;
    int lo;            // the dense range is [lo, pos0)
    int splits, per;   // its splits, and rows per split
    int max_splits;    // at least splits; does not shrink when the range grows
    int merge_heads;   // heads of a group per CTA of the merge
    bool tc;           // the dense range runs on the tensor cores
    float* part;       // records [kv head][query row][split] of hd + 4 floats: max, sum, -, -, o
    float* out;
    int32_t* err;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Dense range on the tensor cores: head sizes it takes, query rows per CTA, cache
// rows per tile, launch.
bool tree_tc_ok(int hd);
__host__ __device__ constexpr int tree_tc_rows(int hd) { return hd > 128 ? 128 : 256; }
__host__ __device__ constexpr int tree_tc_keys(int hd) { return hd > 128 ? 32 : 64; }
cudaError_t tree_tc_launch(const TreeArgs& a, cudaStream_t st);

}  // namespace gncx
