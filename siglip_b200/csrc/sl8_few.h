// sl8_few.h -- sl8_linear_scaled for few rows of A (sl8_few.cu): what the C ABI hands over.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace sl8 {

// Whether these kernels take a product.  Up to 16 rows always; up to 32 and 64 where K is deep enough that the tiles of 64 columns,
// which do not share it out, take longer.
inline bool few_rows(long long M, int K) { return M <= 16 || (M <= 32 && K > 1024) || (M <= 64 && K > 2944); }
constexpr int kFewSplitMax = 8;            // CTAs of a cluster, each with a share of K

struct FewParams {
    int M, N;
    int k_blocks;                    // ceil(K / 128)
    int last_kblock_mmas;            // K = 32 steps of the last one
    const float* row_scales;
    const float* col_scales;
    const void* bias;                // bf16 [N] or fp32 [N] (FLAG_BIAS_F32); may be null
    void* D;
    long long ldd;
    unsigned flags;
    int stages;                      // set by few_launch: depth of the operand ring,
    int share;                       // and rows that each CTA of a cluster finishes (a multiple of four)
    unsigned wait_budget_us;
    uint32_t* status;
};

// Rows of the tile that M rows of A take: the box of map_a.
int few_tile_rows(int M);
// map_b: boxes of 128 rows x 128 bytes of B; map_a: few_tile_rows(M) x 128 bytes of A.
cudaError_t few_launch(bool int8, int sm_count, const CUtensorMap& map_b, const CUtensorMap& map_a, const FewParams& p, cudaStream_t stream);

}  // namespace sl8
