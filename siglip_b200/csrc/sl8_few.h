// sl8_few.h -- sl8_linear_scaled for few rows of A (sl8_few.cu): what the C ABI hands over.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace sl8 {

// Whether these kernels take a product, rather than tiles of 128 x 64 on single CTAs, which do not share out K: the more rows, the
// deeper K has to be.  The rule does not ask for N: with many channels, whose tiles fill the chip, it is up to 3 % off (8 192 x 4 096, 64 rows), and
// with few of them it stops early (4 304 -> 1 152 takes 5.2 us at 64 rows and 7.4 at 65).  us here / on such tiles, int8, by rows:
//   768 x 768     16: 3.0 / 3.4, 32: 3.2 / 3.4, 64: 4.0 / 3.5           4 304 x 1 152  16: 3.8 / 4.7, 32: 4.1 / 4.7, 64: 5.4 / 4.3
//   2 048 x 2 048 32: 4.4 / 4.8, 64: 4.7 / 4.8, 128: 6.6 / 5.0          4 096 x 4 096  16: 6.4 / 10.5, 64: 7.5 / 8.5, 128: 9.6 / 8.9
//   8 192 x 4 096 32: 9.4 / 9.9, 64: 10.4 / 10.1, 128: 12.4 / 10.5      8 192 x 8 192  16: 13.9 / 17.1, 64: 15.5 / 17.6, 128: 17.9 / 18.1
//   4 096 x 8 192 64: 10.3 / 14.4, 128: 12.4 / 14.9                     4 096 x 14 336 16: 12.9 / 23.6, 64: 14.1 / 24, 128: 16.8 / 24.5
inline bool few_rows(long long M, int K) { return M <= 32 || (M <= 64 && K >= 2048) || (M <= 128 && K >= 6144); }
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
