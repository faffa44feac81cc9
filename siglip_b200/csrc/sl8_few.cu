// sl8_few.cu -- sl8_linear_scaled for few rows of A: one token each of some sequences.
//
// What takes time is the weights' way in, so the product is turned round: 128 rows of B are the M of a tcgen05.mma, the rows of A (16,
// 32, 64 or 128, what is missing read as zeros) its N, and a CTA brings 16 KiB of weights per k-block for 2 - 16 KiB of
// activations.  K is shared out to the CTAs of a cluster, because the weights of few output channels would otherwise come through few
// SMs (1 x 4 304 -> 1 152: 8 CTAs 4.0 us, 4 4.4, 2 6.0).  Each CTA writes its partial sums into the shared memory of the one that
// finishes the row, four rows at a time, and one cluster barrier stands between that and the adding up: exact for int8, in the order of
// the ranks for e4m3, so the same result every time.  (Read from there instead, with a barrier on either side: 4.6 us.)
// Bound by the weights' bytes where there are many (32 768 x 4 096, 134 MB: 22.4 us, 6.0 TB/s; 8 192 x 8 192 13.3 us, 5.0), by the way
// of one k-block through all of it where there are few: about 2.8 us from launch to launch (768 x 768).
#include "sl8_kernel.cuh"
#include "sl8_few.h"

namespace sl8 {
namespace {

template <int ROWS>
struct FewTraits {
    static constexpr int W_BYTES = 128 * 128, STAGE_BYTES = W_BYTES + ROWS * 128;
    static constexpr int SUM_BYTES = (ROWS < 4 * kFewSplitMax ? 4 * kFewSplitMax : ROWS) * 128 * 4;   // partial sums of the rows this CTA finishes
    static constexpr int VEC_FLOATS = 2 * 128 + ROWS;                       // column scales, bias, row scales
    // The ring: deep where every CTA has an SM of its own, else such that two CTAs fit one (of 128 rows, one).
    static constexpr int DEEP = ROWS == 128 ? 5 : ROWS == 64 ? 7 : 8, HALF = ROWS == 16 ? 5 : ROWS == 32 ? 4 : ROWS == 64 ? 3 : 5;
    static constexpr int smem_bytes(int stages) { return 1024 + stages * STAGE_BYTES + SUM_BYTES + 4 * VEC_FLOATS + 256; }
    static_assert(smem_bytes(DEEP) <= 232448 && (ROWS == 128 || 2 * (smem_bytes(HALF) + 1024) <= 228 * 1024), "one and two CTAs per SM");
    static_assert(2 * DEEP + 1 <= 32 && 16 * DEEP + 16 <= 256, "a barrier per lane; room for them");
    static constexpr int TMEM_COLS = ROWS < 32 ? 32 : ROWS;
    static_assert(STAGE_BYTES % 1024 == 0, "every operand tile starts on a swizzle-atom boundary");
};

constexpr int kFewThreads = 256;        // two warps for each quarter of the tensor memory's lanes

__device__ __forceinline__ void st_cluster_16(uint32_t addr, float a, float b, float c, float d) {
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(a), "f"(b), "f"(c), "f"(d) : "memory");
}
__device__ __forceinline__ void tmem_ld_32x8(uint32_t taddr, float* v) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
                 : "r"(taddr)
                 : "memory");
}

template <bool I8, int ROWS>
__global__ void __launch_bounds__(kFewThreads) few_rows_kernel(const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_a, const FewParams p) {
    using T = FewTraits<ROWS>;
    extern __shared__ uint8_t few_smem[];
    const uint32_t raw = smem_u32(few_smem);
    const uint32_t base = (raw + 1023u) & ~1023u;
    const uint32_t sums = base + p.stages * T::STAGE_BYTES;                            // [rank][four rows of this CTA][128][4]: 16 bytes per thread, side by side
    float* const vec = reinterpret_cast<float*>(few_smem + (sums - raw) + T::SUM_BYTES);  // column scales, bias, row scales
    uint8_t* const bar_ptr = reinterpret_cast<uint8_t*>(vec + T::VEC_FLOATS);
    const uint32_t full0 = sums + T::SUM_BYTES + 4 * T::VEC_FLOATS, empty0 = full0 + 8 * p.stages, done = empty0 + 8 * p.stages;
    volatile uint32_t* const tmem_ptr = reinterpret_cast<volatile uint32_t*>(bar_ptr + 16 * p.stages + 8);
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

    // No CTA waits for another one of its cluster while it holds tensor memory: that one may itself be waiting for tensor memory, behind a
    // kernel of another stream whose CTAs wait for one another as well (a pair's of the GEMM), and they for what this one holds.  So a CTA says
    // that it runs ahead of the allocation (what another has to know before it writes to its shared memory), and gives the tensor memory
    // back before it waits for the second time.
    if (split > 1) cluster_arrive();
    if (warp == 0) {
        if (lane < 2 * p.stages + 1) {
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
            for (int kb = kb_begin; kb < kb_end && kb < kb_begin + p.stages; kb++) tma_prefetch_l2_2d(&map_b, kb * 128, n0);
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_ptr, 0);
    pdl_wait();
    pdl_release();       // (behind the allocation of tensor memory, on which no later kernel may be ahead of this one)

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
            if (++stage == p.stages) { stage = 0; phase ^= 1u; }
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
            if (++stage == p.stages) { stage = 0; phase ^= 1u; }
        }
    }
    if (warp >= 2) {
        // while the operands come: what the sums are multiplied with
        for (int i = threadIdx.x - 64; i < 128; i += kFewThreads - 64) {
            float col_scale = 0.0f, bias = 0.0f;
            if (n0 + i < p.N) {
                col_scale = ld_f32(p.col_scales + n0 + i);
                if (p.bias) bias = (p.flags & FLAG_BIAS_F32) ? ld_f32(static_cast<const float*>(p.bias) + n0 + i) : ld_bf16(static_cast<const __nv_bfloat16*>(p.bias) + n0 + i);
            }
            vec[i] = col_scale;
            vec[128 + i] = bias;
        }
        for (int i = threadIdx.x - 64; i < p.M; i += kFewThreads - 64) vec[256 + i] = ld_f32(p.row_scales + i);
    }
    __syncthreads();
    const bool ok = __all_sync(0xffffffffu, wait_bar<true>(done, 0, wc, ST_EPI_TMEM_FULL_WAIT, 0)) != 0;
    tc_fence_after();

    const int ch = threadIdx.x & 127, half = threadIdx.x >> 7;       // this thread's output channel (TMEM lane), and which of the rows it takes
    const int n = n0 + ch;
    const float col_scale = vec[ch], bias = vec[128 + ch];
    const auto sum_of = [](float a, float b) { return I8 ? __int_as_float(__float_as_int(a) + __float_as_int(b)) : a + b; };
    const auto number = [](float sum) { return I8 ? __int2float_rn(__float_as_int(sum)) : sum; };
    // rows m .. m + 3 of this channel, as far as there are so many
    const auto finish4 = [&](int m, float s0, float s1, float s2, float s3) {
        const float4 row = *reinterpret_cast<const float4*>(vec + 256 + m);
        float y[4] = {fmaf(number(s0) * row.x, col_scale, bias), fmaf(number(s1) * row.y, col_scale, bias),
                      fmaf(number(s2) * row.z, col_scale, bias), fmaf(number(s3) * row.w, col_scale, bias)};
        if (!(p.flags & FLAG_NO_ACTIVATION)) {
            unpack_f32x2(gelu_tanh_x2(pack_f32x2(y[0], y[1])), y[0], y[1]);
            unpack_f32x2(gelu_tanh_x2(pack_f32x2(y[2], y[3])), y[2], y[3]);
        }
        if (n < p.N) {
            __nv_bfloat16* d = static_cast<__nv_bfloat16*>(p.D) + m * p.ldd + n;
#pragma unroll
            for (int i = 0; i < 4; i++, d += p.ldd)
                if (m + i < p.M) *d = __float2bfloat16_rn(y[i]);
        }
    };
    const uint32_t t_row = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    // the rows of this half, eight or sixteen at a time: f(first row, sums)
    constexpr int CHUNK = ROWS == 16 ? 8 : 16;
    const auto chunks = [&](auto&& f) {
#pragma unroll 1
        for (int c = half * CHUNK; c < p.M; c += 2 * CHUNK) {
            float v[CHUNK];
#pragma unroll
            for (int i = 0; i < CHUNK; i += 8) tmem_ld_32x8(t_row + c + i, v + i);
            tmem_ld_wait();
            f(c, v);
        }
    };
    const auto release = [&]() {
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
        __syncwarp();
    };
    if (split == 1) {
        if (ok)
            chunks([&](int c, const float* v) {
#pragma unroll
                for (int i = 0; i < CHUNK; i += 4)
                    if (c + i < p.M) finish4(c + i, v[i], v[i + 1], v[i + 2], v[i + 3]);
            });
        release();
    } else {
        // Each rank of the cluster finishes `share` rows, a multiple of four: it gets their sums from every rank.
        const int share = p.share, own = static_cast<int>(rank) * share;
        cluster_wait();
        if (ok)
            chunks([&](int c, const float* v) {
                int owner = c / share, at = (c - owner * share) / 4;
#pragma unroll
                for (int i = 0; i < CHUNK; i += 4)
                    if (c + i < p.M) {
                        st_cluster_16(map_to_cta(sums + ((rank * share + 4 * at) * 32 + ch) * 16, owner), v[i], v[i + 1], v[i + 2], v[i + 3]);
                        if (4 * ++at == share) at = 0, owner++;
                    }
            });
        __syncwarp();
        cluster_arrive();
        release();                     // (while the others arrive)
        if (own < p.M) {               // (a CTA that finishes no row is written to by none)
            cluster_wait();
            const float* const mine = reinterpret_cast<const float*>(few_smem + (sums - raw)) + 4 * ch;
            for (int i = 4 * half; i < share && own + i < p.M; i += 8) {
                float4 s = *reinterpret_cast<const float4*>(mine + i * 128);
                for (uint32_t q = 1; q < split; q++) {
                    const float4 o = *reinterpret_cast<const float4*>(mine + (q * share + i) * 128);
                    s = make_float4(sum_of(s.x, o.x), sum_of(s.y, o.y), sum_of(s.z, o.z), sum_of(s.w, o.w));
                }
                finish4(own + i, s.x, s.y, s.z, s.w);
            }
        }
    }
}

// CTAs that share the K of one block of 128 columns: as many as give each SM one, with at least one and a half k-blocks for each.
int blocks_of(int N) { return N / 128 + (N % 128 != 0 ? 1 : 0); }
int few_split(int sm_count, int N, int k_blocks) {
    const int blocks = blocks_of(N);
    int split = 1;
    while (split < kFewSplitMax && blocks * split * 2 <= sm_count && split * 3 <= k_blocks) split *= 2;
    return split;
}

template <bool I8, int ROWS>
cudaError_t launch(FewKernelState& state, int sm_count, const CUtensorMap& map_b, const CUtensorMap& map_a, FewParams p, cudaStream_t stream) {
    int split = few_split(sm_count, p.N, p.k_blocks);
    using T = FewTraits<ROWS>;
    const auto kernel = few_rows_kernel<I8, ROWS>;
    if (!state.attr_set) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, T::smem_bytes(T::DEEP));
        if (e != cudaSuccess) return e;
        state.attr_set = true;
    }
    const int blocks = blocks_of(p.N);
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(kFewThreads, 1, 1);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    const auto shape = [&](int stages) {
        cfg.gridDim = dim3(static_cast<unsigned>(blocks * split), 1, 1);
        cfg.dynamicSmemBytes = static_cast<size_t>(T::smem_bytes(stages));
        attr[0].val.clusterDim.x = static_cast<unsigned>(split);
    };
    // How many clusters of CTAs with the deep ring are resident at once: fewer than the SMs would give room to, because a cluster has
    // to find its SMs in one part of the chip (of eight: 15).
    const auto resident = [&]() {
        int& fit = state.clusters[split == 1 ? 0 : split == 2 ? 1 : split == 4 ? 2 : 3];
        if (fit == 0) {
            shape(T::DEEP);
            cfg.numAttrs = 1;
            if (cudaOccupancyMaxActiveClusters(&fit, kernel, &cfg) != cudaSuccess || fit < 1) {
                (void)cudaGetLastError();
                fit = sm_count / split;
            }
        }
        return fit;
    };
    // The deep ring where all clusters are resident at once with it (1 x 4 096 -> 14 336 12.8 us with two CTAs per SM, 11.7 so).
    // (of 64 and 128 rows a second round of clusters costs more than a share of K twice as long: 64 x 8 192 -> 2 048 11.2 us, 9.8 so)
    while (ROWS >= 64 && split > 1 && blocks > resident()) split /= 2;
    const int most = (p.k_blocks + split - 1) / split;
    p.stages = blocks <= resident() ? T::DEEP : T::HALF;
    if (p.stages > most) p.stages = most;            // (a short ring leaves room for the next kernel's CTAs)
    shape(p.stages);
    cfg.numAttrs = 2;
    p.share = (p.M + 4 * split - 1) / (4 * split) * 4;
    return cudaLaunchKernelEx(&cfg, kernel, map_b, map_a, p);
}

}  // namespace

int few_tile_rows(int M) { return M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : 128; }

cudaError_t few_launch(FewState& state, bool int8, int sm_count, const CUtensorMap& map_b, const CUtensorMap& map_a, const FewParams& p, cudaStream_t stream) {
    const int rows = few_tile_rows(p.M);
    FewKernelState& kernel = state.kernel[int8 ? 1 : 0][rows == 16 ? 0 : rows == 32 ? 1 : rows == 64 ? 2 : 3];
    const auto go = [&](auto f) { return f(kernel, sm_count, map_b, map_a, p, stream); };
    if (int8) return rows == 16 ? go(launch<true, 16>) : rows == 32 ? go(launch<true, 32>) : rows == 64 ? go(launch<true, 64>) : go(launch<true, 128>);
    return rows == 16 ? go(launch<false, 16>) : rows == 32 ? go(launch<false, 32>) : rows == 64 ? go(launch<false, 64>) : go(launch<false, 128>);
}

}  // namespace sl8
