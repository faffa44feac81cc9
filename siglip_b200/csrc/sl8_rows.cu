// sl8_rows.cu -- rows in 8 bits with a scale of their own (include/siglip_fp8.h): sl8_quantize_rows and sl8_rmsnorm_quantize,
// the operands of sl8_linear_scaled.
#include <cuda_bf16.h>

#include "sl8_internal.h"

namespace {

typedef __nv_bfloat16 bf16;

struct RowArgs {
    const void* x;        long long ld;
    const void* residual; long long ld_res;      // may be null
    void* sum;            long long ld_sum;      // x + residual, with a residual only; may be x or residual
    const float* gamma;                          // null = 1
    float eps;
    const float* scale;                          // one scale for all rows (row_scales null); null = 1
    uint8_t* out;         long long ld_out;
    float* row_scales;                           // a scale per row, or null
    long long rows;
    int cols;
    int int8;                                    // codes: int8, else e4m3
};

// ---- eight consecutive elements as they lie in memory, and their values
template <typename T>
struct Eight {
    uint32_t w[2 * sizeof(T)];
};
__device__ __forceinline__ uint16_t ld_u16(const void* p) {
    uint16_t v;
    asm volatile("ld.global.u16 %0, [%1];" : "=h"(v) : "l"(p) : "memory");
    return v;
}
// `have` of them; VEC: all eight, from a 16-byte boundary.
template <bool VEC, typename T>
__device__ __forceinline__ void fetch(Eight<T>& e, const T* p, int have) {
    if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++) {
            const uint4 q = sl8::ld_16(p + i * (16 / (int)sizeof(T)));
            e.w[4 * i] = q.x; e.w[4 * i + 1] = q.y; e.w[4 * i + 2] = q.z; e.w[4 * i + 3] = q.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            if constexpr (sizeof(T) == 4) {
                e.w[i] = i < have ? __float_as_uint(sl8::ld_f32(p + i)) : 0u;
            } else {
                const uint32_t b = i < have ? ld_u16(p + i) : 0u;
                if (i & 1) e.w[i / 2] |= b << 16;
                else e.w[i / 2] = b;
            }
        }
    }
}
template <typename T>
__device__ __forceinline__ float value(const Eight<T>& e, int i) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(e.w[i]);
    else return (i & 1) ? sl8::bf16_hi_f32(e.w[i / 2]) : sl8::bf16_lo_f32(e.w[i / 2]);
}
template <bool VEC, typename T>
__device__ __forceinline__ void put_sum(T* p, const float (&v)[8], int have) {
    if constexpr (sizeof(T) == 4) {
        if constexpr (VEC) {
            reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
            reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (i < have) p[i] = v[i];
        }
    } else {
        if constexpr (VEC) {
            *reinterpret_cast<uint4*>(p) = make_uint4(sl8::pack_bf16x2(v[0], v[1]), sl8::pack_bf16x2(v[2], v[3]),
                                                      sl8::pack_bf16x2(v[4], v[5]), sl8::pack_bf16x2(v[6], v[7]));
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (i < have) p[i] = __float2bfloat16_rn(v[i]);
        }
    }
}

// Four int8 codes: y * inv + 1.5 * 2^23 leaves round-to-nearest-even(y * inv) in the low byte (|y * inv| <= 127).
__device__ __forceinline__ uint32_t int8x4(float a, float b, float c, float d, float inv) {
    constexpr float M = 12582912.0f;
    const uint32_t p = __float_as_uint(fmaf(a, inv, M)), q = __float_as_uint(fmaf(b, inv, M));
    const uint32_t r = __float_as_uint(fmaf(c, inv, M)), s = __float_as_uint(fmaf(d, inv, M));
    return __byte_perm(__byte_perm(p, q, 0x0040), __byte_perm(r, s, 0x0040), 0x5410);
}
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d, float inv) {
    return static_cast<uint32_t>(sl8::pack_e4m3x2(a * inv, b * inv)) | (static_cast<uint32_t>(sl8::pack_e4m3x2(c * inv, d * inv)) << 16);
}
template <bool VEC>
__device__ __forceinline__ void put_codes(uint8_t* p, const float (&y)[8], float inv, bool int8, int have) {
    const uint32_t lo = int8 ? int8x4(y[0], y[1], y[2], y[3], inv) : e4m3x4(y[0], y[1], y[2], y[3], inv);
    const uint32_t hi = int8 ? int8x4(y[4], y[5], y[6], y[7], inv) : e4m3x4(y[4], y[5], y[6], y[7], inv);
    if constexpr (VEC) {
        *reinterpret_cast<uint2*>(p) = make_uint2(lo, hi);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i < have) p[i] = static_cast<uint8_t>((i < 4 ? lo : hi) >> (8 * (i & 3)));
    }
}

// |v| as an integer: ordered like the numbers, infinity above them and NaN above that, so that none gets lost in a maximum.
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

struct Stats {
    float squares;        // sum of h^2
    uint32_t largest;     // magnitude of the largest h * gamma
};
template <bool NORM>
__device__ __forceinline__ Stats reduce_warp(Stats s) {
    if constexpr (NORM) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s.squares += __shfl_xor_sync(0xffffffffu, s.squares, o);
    }
    s.largest = __reduce_max_sync(0xffffffffu, s.largest);
    return s;
}
// Over the G threads of a row; `turn` counts the calls (the rows of a block use two sets of partial results in turn, so one barrier does).
template <bool NORM, int G>
__device__ __forceinline__ Stats reduce(Stats s, int turn) {
    s = reduce_warp<NORM>(s);
    if constexpr (G > 32) {
        __shared__ Stats part[2][G / 32];
        if ((threadIdx.x & 31) == 0) part[turn & 1][threadIdx.x >> 5] = s;
        __syncthreads();
        s = part[turn & 1][0];
#pragma unroll
        for (int i = 1; i < G / 32; i++) {
            const Stats o = part[turn & 1][i];
            s.squares += o.squares;
            s.largest = max(s.largest, o.largest);
        }
    }
    return s;
}

// What a row's codes are multiples of, and its reciprocal.
struct Scaling {
    float rstd, scale, inv;
};
template <bool NORM>
__device__ __forceinline__ Scaling scaling(const RowArgs& a, const Stats& s, float inv_n, float given_inv) {
    Scaling r;
    // a sum of squares that is no number (an infinity or NaN among the elements, or squares beyond fp32): nothing that comes out is one
    r.rstd = !NORM ? 1.0f : s.squares < __int_as_float(0x7F800000) ? rsqrtf(fmaf(s.squares, inv_n, a.eps)) : __int_as_float(0x7FC00000);
    r.scale = 0.0f;
    r.inv = given_inv;
    if (a.row_scales) {
        // rounding is monotonic: the largest |h * gamma| times rstd is the largest |h * gamma * rstd|
        const float largest = __uint_as_float(s.largest) * r.rstd;
        if (largest == 0.0f) r.scale = 1.0f;
        else if (largest < __int_as_float(0x7F800000)) r.scale = fmaxf(__fdiv_rn(largest, a.int8 ? 127.0f : 448.0f), 1.17549435e-38f);
        else r.scale = __int_as_float(0x7FC00000);
        r.inv = __frcp_rn(r.scale);
    }
    return r;
}

constexpr int kRowThreads = 128;

// A row by G threads, CH groups of eight elements each, read once and held in registers; statistics in fp32.  Bound by the bytes of
// x, the residual, their sum and the codes.
template <typename T, bool NORM, bool VEC, int G, int CH>
__global__ void __launch_bounds__(G < kRowThreads ? kRowThreads : G) row_kernel(const RowArgs a) {
    constexpr int BLOCK = G < kRowThreads ? kRowThreads : G, ROWS = BLOCK / G;
    const int c0 = (threadIdx.x % G) * 8;
    const float inv_n = 1.0f / static_cast<float>(a.cols);
    sl8::pdl_wait();
    sl8::pdl_release();
    const float given_inv = a.row_scales ? 0.0f : __frcp_rn(a.scale ? sl8::ld_f32(a.scale) : 1.0f);
    int turn = 0;
    for (long long r = static_cast<long long>(blockIdx.x) * ROWS + threadIdx.x / G; r < a.rows; r += static_cast<long long>(gridDim.x) * ROWS, turn++) {
        const T* const x = static_cast<const T*>(a.x) + r * a.ld;
        float v[CH][8];
        {
            Eight<T> e[CH];
#pragma unroll
            for (int j = 0; j < CH; j++)
                if (c0 + 8 * G * j < a.cols) fetch<VEC>(e[j], x + c0 + 8 * G * j, a.cols - (c0 + 8 * G * j));
            if (NORM && a.residual) {
                const T* const res = static_cast<const T*>(a.residual) + r * a.ld_res;
                T* const sum = static_cast<T*>(a.sum) + r * a.ld_sum;
                Eight<T> f[CH];
#pragma unroll
                for (int j = 0; j < CH; j++)
                    if (c0 + 8 * G * j < a.cols) fetch<VEC>(f[j], res + c0 + 8 * G * j, a.cols - (c0 + 8 * G * j));
#pragma unroll
                for (int j = 0; j < CH; j++)
                    if (c0 + 8 * G * j < a.cols) {
#pragma unroll
                        for (int i = 0; i < 8; i++) v[j][i] = value(e[j], i) + value(f[j], i);
                        put_sum<VEC>(sum + c0 + 8 * G * j, v[j], a.cols - (c0 + 8 * G * j));
                    }
            } else {
#pragma unroll
                for (int j = 0; j < CH; j++)
#pragma unroll
                    for (int i = 0; i < 8; i++) v[j][i] = value(e[j], i);
            }
        }
        Stats s = {0.0f, 0u};
#pragma unroll
        for (int j = 0; j < CH; j++)
            if (c0 + 8 * G * j < a.cols) {
                if constexpr (NORM) {
#pragma unroll
                    for (int i = 0; i < 8; i++) s.squares = fmaf(v[j][i], v[j][i], s.squares);
                    if (a.gamma) {
                        Eight<float> g;
                        fetch<VEC>(g, a.gamma + c0 + 8 * G * j, a.cols - (c0 + 8 * G * j));
#pragma unroll
                        for (int i = 0; i < 8; i++) v[j][i] *= value(g, i);
                    }
                }
#pragma unroll
                for (int i = 0; i < 8; i++) s.largest = max(s.largest, magnitude(v[j][i]));
            }
        const Scaling k = scaling<NORM>(a, reduce<NORM, G>(s, turn), inv_n, given_inv);
        uint8_t* const out = a.out + r * a.ld_out;
#pragma unroll
        for (int j = 0; j < CH; j++)
            if (c0 + 8 * G * j < a.cols) {
                if constexpr (NORM) {
#pragma unroll
                    for (int i = 0; i < 8; i++) v[j][i] *= k.rstd;
                }
                put_codes<VEC>(out + c0 + 8 * G * j, v[j], k.inv, a.int8 != 0, a.cols - (c0 + 8 * G * j));
            }
        if (a.row_scales && threadIdx.x % G == 0) a.row_scales[r] = k.scale;
    }
}

// Rows too long for the registers of a block: read twice, statistics first.  The sum is written the second time only, because it may
// lie where the first reading still has to find x or the residual.
constexpr int kLongThreads = 512;
template <typename T, bool NORM, bool VEC>
__global__ void __launch_bounds__(kLongThreads) long_row_kernel(const RowArgs a) {
    const float inv_n = 1.0f / static_cast<float>(a.cols);
    sl8::pdl_wait();
    sl8::pdl_release();
    const float given_inv = a.row_scales ? 0.0f : __frcp_rn(a.scale ? sl8::ld_f32(a.scale) : 1.0f);
    int turn = 0;
    for (long long r = blockIdx.x; r < a.rows; r += gridDim.x, turn++) {
        const T* const x = static_cast<const T*>(a.x) + r * a.ld;
        const T* const res = NORM && a.residual ? static_cast<const T*>(a.residual) + r * a.ld_res : nullptr;
        T* const sum = static_cast<T*>(a.sum) + r * a.ld_sum;
        const auto load = [&](int c, float (&v)[8], bool write) {
            Eight<T> e;
            fetch<VEC>(e, x + c, a.cols - c);
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = value(e, i);
            if (res) {
                fetch<VEC>(e, res + c, a.cols - c);
#pragma unroll
                for (int i = 0; i < 8; i++) v[i] += value(e, i);
                if (write) put_sum<VEC>(sum + c, v, a.cols - c);
            }
        };
        const auto times_gamma = [&](int c, float (&v)[8]) {
            if (NORM && a.gamma) {
                Eight<float> g;
                fetch<VEC>(g, a.gamma + c, a.cols - c);
#pragma unroll
                for (int i = 0; i < 8; i++) v[i] *= value(g, i);
            }
        };
        Stats s = {0.0f, 0u};
        for (int c = threadIdx.x * 8; c < a.cols; c += 8 * kLongThreads) {
            float v[8];
            load(c, v, false);
            if constexpr (NORM) {
#pragma unroll
                for (int i = 0; i < 8; i++) s.squares = fmaf(v[i], v[i], s.squares);
                times_gamma(c, v);
            }
#pragma unroll
            for (int i = 0; i < 8; i++) s.largest = max(s.largest, magnitude(v[i]));
        }
        const Scaling k = scaling<NORM>(a, reduce<NORM, kLongThreads>(s, turn), inv_n, given_inv);
        for (int c = threadIdx.x * 8; c < a.cols; c += 8 * kLongThreads) {
            float v[8];
            load(c, v, true);
            if constexpr (NORM) {
                times_gamma(c, v);
#pragma unroll
                for (int i = 0; i < 8; i++) v[i] *= k.rstd;
            }
            put_codes<VEC>(a.out + r * a.ld_out + c, v, k.inv, a.int8 != 0, a.cols - c);
        }
        if (a.row_scales && threadIdx.x == 0) a.row_scales[r] = k.scale;
    }
}

template <typename T, bool NORM, bool VEC>
cudaError_t launch_rows(int sm_count, cudaStream_t s, const RowArgs& a) {
    const auto go = [&](auto kernel, int g, int threads, int per_sm) {
        const long long want = (a.rows + threads / g - 1) / (threads / g), cap = static_cast<long long>(sm_count) * per_sm;
        return sl8_launch_chained(kernel, static_cast<unsigned>(want < cap ? want : cap), threads, 0, s, a);
    };
#define SL8_ROWS(G, CH, PER_SM) go(row_kernel<T, NORM, VEC, G, CH>, G, G < kRowThreads ? kRowThreads : G, PER_SM)
    if (a.cols <= 256) return SL8_ROWS(32, 1, 32);
    if (a.cols <= 768) return SL8_ROWS(32, 3, 32);
    if (a.cols <= 1280) return SL8_ROWS(32, 5, 32);
    if (a.cols <= 2048) return SL8_ROWS(128, 2, 32);
    if (a.cols <= 4096) return SL8_ROWS(128, 4, 32);
    if (a.cols <= 8192) return SL8_ROWS(256, 4, 16);
    if (a.cols <= 16384) return SL8_ROWS(512, 4, 8);
#undef SL8_ROWS
    return go(long_row_kernel<T, NORM, VEC>, kLongThreads, kLongThreads, 8);
}

template <typename T, bool NORM>
int run_rows(sl8_handle_t h, const RowArgs& a, sl8_stream_t stream, const char* what) {
    Sl8DeviceGuard guard(h->device);
    if (!guard.ok) return sl8_fail(h, SL8_ERR_CUDA, "cudaSetDevice failed");
    constexpr int PER_16 = 16 / sizeof(T);
    // eight elements per access where every row allows it, element by element otherwise
    const bool vec = a.cols % 8 == 0 && sl8_aligned16(a.x) && a.ld % PER_16 == 0 && a.ld_out % 8 == 0 && (reinterpret_cast<uintptr_t>(a.out) & 7u) == 0 &&
                     (!a.gamma || sl8_aligned16(a.gamma)) &&
                     (!a.residual || (sl8_aligned16(a.residual) && a.ld_res % PER_16 == 0 && sl8_aligned16(a.sum) && a.ld_sum % PER_16 == 0));
    const cudaError_t e = vec ? launch_rows<T, NORM, true>(h->sm_count, static_cast<cudaStream_t>(stream), a)
                              : launch_rows<T, NORM, false>(h->sm_count, static_cast<cudaStream_t>(stream), a);
    return e == cudaSuccess ? SL8_OK : sl8_fail_cuda(h, e, what);
}

bool element_aligned(const void* p, int dtype) { return (reinterpret_cast<uintptr_t>(p) & (dtype == SL8_DT_F32 ? 3u : 1u)) == 0; }
bool float_aligned(const float* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

}  // namespace

SL8_API int sl8_quantize_rows(sl8_handle_t h, const void* x, int dtype, int64_t rows, int cols, int64_t ld, int code_type, void* out,
                              int64_t ld_out, float* row_scales, sl8_stream_t stream) {
    if (!h) return SL8_ERR_INVALID_VALUE;
    if (!x || !out || !row_scales || rows < 1 || cols < 1 || ld < cols || ld_out < cols)
        return sl8_fail(h, SL8_ERR_INVALID_VALUE, "bad quantize_rows arguments");
    if (dtype != SL8_DT_F32 && dtype != SL8_DT_BF16) return sl8_fail(h, SL8_ERR_INVALID_VALUE, "unknown dtype");
    if (code_type != SL8_CODE_INT8 && code_type != SL8_CODE_E4M3) return sl8_fail(h, SL8_ERR_INVALID_VALUE, "unknown code type");
    if (!element_aligned(x, dtype) || !float_aligned(row_scales)) return sl8_fail(h, SL8_ERR_ALIGNMENT, "x and row_scales must be aligned to their elements");
    RowArgs a = {};
    a.x = x; a.ld = ld;
    a.out = static_cast<uint8_t*>(out); a.ld_out = ld_out;
    a.row_scales = row_scales; a.rows = rows; a.cols = cols; a.int8 = code_type == SL8_CODE_INT8;
    return dtype == SL8_DT_F32 ? run_rows<float, false>(h, a, stream, "quantize_rows kernel launch") : run_rows<bf16, false>(h, a, stream, "quantize_rows kernel launch");
}

SL8_API int sl8_rmsnorm_quantize(sl8_handle_t h, const void* x, int dtype, int64_t rows, int cols, int64_t ld, const void* residual,
                                 int64_t ld_res, void* sum, int64_t ld_sum, const float* gamma, float eps, int code_type, const float* scale,
                                 void* out, int64_t ld_out, float* row_scales, sl8_stream_t stream) {
    if (!h) return SL8_ERR_INVALID_VALUE;
    if (!x || !out || rows < 1 || cols < 1 || ld < cols || ld_out < cols || !(eps >= 0.0f))
        return sl8_fail(h, SL8_ERR_INVALID_VALUE, "bad rmsnorm arguments");
    if (dtype != SL8_DT_F32 && dtype != SL8_DT_BF16) return sl8_fail(h, SL8_ERR_INVALID_VALUE, "unknown dtype");
    if (code_type != SL8_CODE_INT8 && code_type != SL8_CODE_E4M3) return sl8_fail(h, SL8_ERR_INVALID_VALUE, "unknown code type");
    if ((residual == nullptr) != (sum == nullptr)) return sl8_fail(h, SL8_ERR_INVALID_VALUE, "residual and sum come together");
    if (residual && (ld_res < cols || ld_sum < cols)) return sl8_fail(h, SL8_ERR_INVALID_VALUE, "ld_res / ld_sum smaller than cols");
    if (row_scales && scale) return sl8_fail(h, SL8_ERR_INVALID_VALUE, "a scale is given, or written for each row");
    if (!row_scales && code_type == SL8_CODE_INT8) return sl8_fail(h, SL8_ERR_INVALID_VALUE, "int8 codes have a scale for each row");
    if (!element_aligned(x, dtype) || !element_aligned(residual, dtype) || !element_aligned(sum, dtype) || !float_aligned(gamma) ||
        !float_aligned(scale) || !float_aligned(row_scales))
        return sl8_fail(h, SL8_ERR_ALIGNMENT, "x, residual, sum, gamma and the scales must be aligned to their elements");
    RowArgs a = {};
    a.x = x; a.ld = ld;
    a.residual = residual; a.ld_res = ld_res; a.sum = sum; a.ld_sum = ld_sum;
    a.gamma = gamma; a.eps = eps; a.scale = scale;
    a.out = static_cast<uint8_t*>(out); a.ld_out = ld_out;
    a.row_scales = row_scales; a.rows = rows; a.cols = cols; a.int8 = code_type == SL8_CODE_INT8;
    return dtype == SL8_DT_F32 ? run_rows<float, true>(h, a, stream, "rmsnorm kernel launch") : run_rows<bf16, true>(h, a, stream, "rmsnorm kernel launch");
}
