// sl8_few.h -- sl8_linear_scaled for few rows of A (sl8_few.cu): what the C ABI hands over.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace sl8 {

// Whether these kernels take a product, rather than tiles of 128 x 64 on single CTAs, which do not share out K: up to 16 rows always; from
// there on the partial sums that change hands cost 50 - 100 ns a row, which only a deep K pays for.  us here / on such tiles, int8:
//   16 rows: 768 x 768 2.9 / 3.4, 4 304 x 1 152 3.9 / 4.8, 4 096 x 4 096 6.4 / 10.5, 14 336 x 4 096 12.3 / 26
//   32: 768 x 768 3.5 / 3.4, 4 304 x 1 152 4.75 / 4.8, 1 152 x 4 304 4.65 / 6.9, 4 096 x 4 096 7.4 / 8.4
//   64: 4 304 x 1 152 5.3 / 4.4, 1 152 x 4 304 7.0 / 7.1, 4 096 x 4 096 8.7 / 8.6, 14 336 x 4 096 13.2 / 16.6, 4 096 x 14 336 15.3 / 24
//   128: 4 096 x 4 096 13.9 / 8.8, 4 096 x 8 192 16.8 / 14.9, 4 096 x 14 336 21 / 24.6, 1 024 x 16 384 14.7 / 20.5
inline bool few_rows(long long M, int K) { return M <= 16 || (M <= 32 && K > 1024) || (M <= 64 && K > 2944) || (M <= 128 && K >= 12288); }
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

// What a handle remembers of them.
struct FewKernelState {
    bool attr_set = false;
    int clusters[4] = {};            // resident at once, by the CTAs of a cluster: 1, 2, 4, 8
};
struct FewState {
    FewKernelState kernel[2][4];     // e4m3, int8; 16, 32, 64, 128 rows
};
// Rows of the tile that M rows of A take: the box of map_a.
int few_tile_rows(int M);
// map_b: boxes of 128 rows x 128 bytes of B; map_a: few_tile_rows(M) x 128 bytes of A.
cudaError_t few_launch(FewState& state, bool int8, int sm_count, const CUtensorMap& map_b, const CUtensorMap& map_a, const FewParams& p, cudaStream_t stream);

}  // namespace sl8
