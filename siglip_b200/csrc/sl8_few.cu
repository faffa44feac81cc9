// sl8_few.cu -- sl8_linear_scaled for few rows of A: one token each of some sequences.
//
// The product is that of the weights' bytes with hardly anything, so it is turned round: 128 rows of B are the M of a
// tcgen05.mma, the rows of A (16, 32 or 64, what is missing read as zeros) its N, and a CTA brings 16 KiB of weights per k-block
// for 2 - 8 KiB of activations.  K is shared by the CTAs of a cluster, because the weights of few output channels would
// otherwise come through few SMs; their partial sums meet in shared memory (exact for int8, in the order of the ranks for
// e4m3: the same result every time), and each CTA finishes a share of the rows.
#include "sl8_kernel.cuh"
#include "sl8_few.h"

namespace sl8 {
namespace {

template <int ROWS>
struct FewTraits {
    static constexpr int W_BYTES = 128 * 128, STAGE_BYTES = W_BYTES + ROWS * 128;
    static constexpr int STAGES = ROWS == 16 ? 6 : ROWS == 32 ? 5 : 4;      // about 100 KiB: two CTAs fit an SM
    static constexpr int SMEM_BYTES = 1024 + STAGES * STAGE_BYTES + 256;
    static constexpr int TMEM_COLS = ROWS < 32 ? 32 : ROWS;
    static_assert(STAGE_BYTES % 1024 == 0, "every operand tile starts on a swizzle-atom boundary");
    static_assert(ROWS * 128 * 4 <= STAGES * STAGE_BYTES, "partial sums fit where the operands were");
};

constexpr int kFewThreads = 128;

__device__ __forceinline__ uint32_t ld_cluster(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void sts32(uint32_t addr, uint32_t v) { asm volatile("st.shared.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }

template <bool I8, int ROWS>
__global__ void __launch_bounds__(kFewThreads) few_rows_kernel(const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_a, const FewParams p) {
    using T = FewTraits<ROWS>;
    extern __shared__ uint8_t few_smem[];
    const uint32_t raw = smem_u32(few_smem);
    const uint32_t base = (raw + 1023u) & ~1023u;
    uint8_t* const bar_ptr = few_smem + (base - raw) + T::STAGES * T::STAGE_BYTES;
    const uint32_t full0 = base + T::STAGES * T::STAGE_BYTES, empty0 = full0 + 8 * T::STAGES, done = empty0 + 8 * T::STAGES;
    volatile uint32_t* const tmem_ptr = reinterpret_cast<volatile uint32_t*>(bar_ptr + 16 * T::STAGES + 8);
    volatile uint32_t* const abort_flag = tmem_ptr + 1;

    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    uint32_t split;
    asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(split));
    const uint32_t rank = cluster_ctarank();
    const int n0 = static_cast<int>(blockIdx.x / split) * 128;
    const int kb_begin = static_cast<int>(p.k_blocks * rank / split), kb_end = static_cast<int>(p.k_blocks * (rank + 1) / split);

    WaitCtx wc;
    wc.abort_flag = abort_flag;
    wc.status = p.status;
    wc.budget_ns = static_cast<unsigned long long>(p.wait_budget_us) * 1000ull;
    wc.peer_abort = 0u;              // (the other CTAs of the cluster wait for nothing but its barriers, which every CTA reaches)
    wc.tile = blockIdx.x / split;

    if (warp == 0) {
        if (lane < 2 * T::STAGES + 1) {
            mbar_init(full0 + 8 * lane, 1);
            fence_mbar_init();
        }
        if (lane == 0) *abort_flag = 0u;
    } else if (warp == 1) {
        tmem_alloc<1>(smem_u32(const_cast<uint32_t*>(tmem_ptr)), T::TMEM_COLS);
        tmem_relinquish<1>();
    } else if (warp == 2) {
        if (elect_one()) {
            prefetch_tensormap(&map_b);
            prefetch_tensormap(&map_a);
            // (weights on their way into L2 while the kernel ahead finishes: a hint, like that of the other GEMMs)
            for (int kb = kb_begin; kb < kb_end && kb < kb_begin + T::STAGES; kb++) tma_prefetch_l2_2d(&map_b, kb * 128, n0);
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_ptr, 0);
    pdl_wait();
    pdl_release();       // (behind the allocation of tensor memory, on which no later kernel may be ahead of this one)

    const int n = n0 + static_cast<int>(threadIdx.x);       // this thread's output channel: TMEM lane threadIdx.x
    float col_scale = 0.0f, bias = 0.0f;
    if (n < p.N) {
        col_scale = ld_f32(p.col_scales + n);
        if (p.bias) bias = (p.flags & FLAG_BIAS_F32) ? ld_f32(static_cast<const float*>(p.bias) + n) : ld_bf16(static_cast<const __nv_bfloat16*>(p.bias) + n);
    }

    if (warp == 0) {
        int stage = 0;
        uint32_t phase = 0;
        for (int kb = kb_begin; kb < kb_end; kb++) {
            if (__all_sync(0xffffffffu, wait_bar<true>(empty0 + 8 * stage, phase ^ 1u, wc, ST_PRODUCER_EMPTY_WAIT, stage)) == 0) break;
            if (elect_one()) {
                const uint32_t dst = base + stage * T::STAGE_BYTES, bar = full0 + 8 * stage;
                mbar_arrive_expect_tx(bar, T::STAGE_BYTES);
                // (test aid: the activations of a share's second k-block are never brought)
                if (!((p.flags & FLAG_TEST_DROP_B) && kb == kb_begin + 1)) tma_load_2d(dst + T::W_BYTES, &map_a, kb * 128, 0, bar);
                tma_load_2d(dst, &map_b, kb * 128, n0, bar);
            }
            __syncwarp();
            if (++stage == T::STAGES) { stage = 0; phase ^= 1u; }
        }
    } else if (warp == 1) {
        const uint32_t idesc = I8 ? make_idesc_i8_s32(128, ROWS) : make_idesc_e4m3_f32(128, ROWS);
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int kb = kb_begin; kb < kb_end; kb++) {
            ok = __all_sync(0xffffffffu, wait_bar<true>(full0 + 8 * stage, phase, wc, ST_MMA_FULL_WAIT, stage)) != 0;
            if (!ok) break;
            tc_fence_after();
            if (elect_one()) {
                const uint32_t at = base + stage * T::STAGE_BYTES;
                const uint64_t wdesc = make_kmajor_sw128_desc(at), xdesc = make_kmajor_sw128_desc(at + T::W_BYTES);
                const int steps = kb == p.k_blocks - 1 ? p.last_kblock_mmas : 4;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    if (j < steps) {
                        if constexpr (I8) mma_i8<1>(tmem, wdesc + 2 * j, xdesc + 2 * j, idesc, (kb != kb_begin || j != 0) ? 1u : 0u);
                        else mma_f8<1>(tmem, wdesc + 2 * j, xdesc + 2 * j, idesc, (kb != kb_begin || j != 0) ? 1u : 0u);
                    }
                }
                mma_commit(empty0 + 8 * stage);
                if (kb == kb_end - 1) mma_commit(done);
            }
            __syncwarp();
            if (++stage == T::STAGES) { stage = 0; phase ^= 1u; }
        }
    }
    __syncwarp();
    const bool ok = __all_sync(0xffffffffu, wait_bar(done, 0, wc, ST_EPI_TMEM_FULL_WAIT, 0)) != 0;
    tc_fence_after();

    const auto sum_of = [](uint32_t a, uint32_t b) { return I8 ? a + b : __float_as_uint(__uint_as_float(a) + __uint_as_float(b)); };
    const auto finish = [&](int m, uint32_t sum) {
        const float acc = I8 ? __int2float_rn(static_cast<int>(sum)) : __uint_as_float(sum);
        float y = fmaf(acc * ld_f32(p.row_scales + m), col_scale, bias);
        if (!(p.flags & FLAG_NO_ACTIVATION)) {
            float unused;
            unpack_f32x2(gelu_tanh_x2(pack_f32x2(y, 0.0f)), y, unused);
        }
        if (n < p.N) static_cast<__nv_bfloat16*>(p.D)[m * p.ldd + n] = __float2bfloat16_rn(y);
    };
    const uint32_t t_row = tmem + (static_cast<uint32_t>(warp * 32) << 16);
    if (split == 1) {
        if (ok) {
#pragma unroll 1
            for (int c = 0; c < p.M; c += 32) {
                float v[32];
                tmem_ld_32x32(t_row + c, v);       // (of 16 rows: with 16 columns that nothing wrote and nothing uses)
                tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 32; i++)
                    if (c + i < p.M) finish(c + i, __float_as_uint(v[i]));
            }
        }
    } else {
        // Sums of row m, column n0 + i: at base + (m * 128 + i) * 4, where the operands were (every copy has landed and been read).
        const uint32_t mine = base + 4 * threadIdx.x;
        if (ok) {
#pragma unroll 1
            for (int c = 0; c < p.M; c += 32) {
                float v[32];
                tmem_ld_32x32(t_row + c, v);
                tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 32; i++)
                    if (c + i < p.M) sts32(mine + (c + i) * 512, __float_as_uint(v[i]));
            }
        }
        __syncwarp();
        cluster_arrive();
        cluster_wait();
        const int m_end = static_cast<int>(p.M * (rank + 1) / split);
        for (int m = static_cast<int>(p.M * rank / split); m < m_end; m++) {
            uint32_t part[kFewSplitMax];
#pragma unroll
            for (int q = 0; q < kFewSplitMax; q++)
                if (q < static_cast<int>(split)) part[q] = ld_cluster(map_to_cta(mine + m * 512, q));
            uint32_t sum = part[0];
#pragma unroll
            for (int q = 1; q < kFewSplitMax; q++)
                if (q < static_cast<int>(split)) sum = sum_of(sum, part[q]);
            finish(m, sum);
        }
        __syncwarp();
        cluster_arrive();
        cluster_wait();        // its sums have been read
    }

    tc_fence_before();
    __syncthreads();
    if (*abort_flag) {         // copies and MMAs in flight land before their memory is released
        const unsigned long long t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 200000ull) {
        }
        __syncthreads();
    }
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc<1>(tmem, T::TMEM_COLS);
    }
}

template <bool I8, int ROWS>
cudaError_t launch(int split, const CUtensorMap& map_b, const CUtensorMap& map_a, const FewParams& p, cudaStream_t stream) {
    using T = FewTraits<ROWS>;
    const auto kernel = few_rows_kernel<I8, ROWS>;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, T::SMEM_BYTES);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>((p.N + 127) / 128 * split), 1, 1);
    cfg.blockDim = dim3(kFewThreads, 1, 1);
    cfg.dynamicSmemBytes = T::SMEM_BYTES;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(split);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kernel, map_b, map_a, p);
}

}  // namespace

int few_tile_rows(int M) { return M <= 16 ? 16 : M <= 32 ? 32 : 64; }

int few_split(int sm_count, int N, int k_blocks) {
    const int blocks = (N + 127) / 128;
    int split = 1;
    while (split < kFewSplitMax && blocks * split * 2 <= 2 * sm_count && split * 4 <= k_blocks) split *= 2;
    return split;
}

cudaError_t few_launch(bool int8, int split, const CUtensorMap& map_b, const CUtensorMap& map_a, const FewParams& p, cudaStream_t stream) {
    const int rows = few_tile_rows(p.M);
    if (int8) return rows == 16 ? launch<true, 16>(split, map_b, map_a, p, stream) : rows == 32 ? launch<true, 32>(split, map_b, map_a, p, stream) : launch<true, 64>(split, map_b, map_a, p, stream);
    return rows == 16 ? launch<false, 16>(split, map_b, map_a, p, stream) : rows == 32 ? launch<false, 32>(split, map_b, map_a, p, stream) : launch<false, 64>(split, map_b, map_a, p, stream);
}

}  // namespace sl8
