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
    uint32_t* status;                            // bounded waits, as in the GEMMs
    unsigned wait_budget_us;
    int drop;                                    // test aid: the copy of row 1 is never issued
};

// ---- eight elements of a row as they lie in memory, and their values
template <typename T>
struct Eight {
    uint32_t w[2 * sizeof(T)];
};
__device__ __forceinline__ uint16_t ld_u16(const void* p) {
    uint16_t v;
    asm volatile("ld.global.u16 %0, [%1];" : "=h"(v) : "l"(p) : "memory");
    return v;
}
// VEC: eight in a row from a 16-byte boundary.  Otherwise every 32nd, so that the lanes of a warp read consecutive elements: a warp has
// the same 256 of a row either way.  `left`: elements from the first of the eight to the row's end; the ones beyond are zero (the
// last of the row is read in their place: no load waits for a condition on another).
template <bool VEC, typename T>
__device__ __forceinline__ void fetch(Eight<T>& e, const T* p, int left) {
    if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++) {
            const uint4 q = sl8::ld_16(p + i * (16 / (int)sizeof(T)));
            e.w[4 * i] = q.x; e.w[4 * i + 1] = q.y; e.w[4 * i + 2] = q.z; e.w[4 * i + 3] = q.w;
        }
    } else {
        const auto put = [&](int i, const T* at, bool inside) {
            uint32_t b;
            if constexpr (sizeof(T) == 4) b = __float_as_uint(sl8::ld_f32(at));
            else b = ld_u16(at);
            if (!inside) b = 0u;
            if constexpr (sizeof(T) == 4) e.w[i] = b;
            else if (i & 1) e.w[i / 2] |= b << 16;
            else e.w[i / 2] = b;
        };
        if (left > 224) {
#pragma unroll
            for (int i = 0; i < 8; i++) put(i, p + 32 * i, true);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) put(i, p + min(32 * i, left - 1), 32 * i < left);
        }
    }
}
template <typename T>
__device__ __forceinline__ float value(const Eight<T>& e, int i) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(e.w[i]);
    else return (i & 1) ? sl8::bf16_hi_f32(e.w[i / 2]) : sl8::bf16_lo_f32(e.w[i / 2]);
}
template <bool VEC, typename T>
__device__ __forceinline__ void put_sum(T* p, const float (&v)[8], int left) {
    if constexpr (VEC && sizeof(T) == 4) {
        reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else if constexpr (VEC) {
        *reinterpret_cast<uint4*>(p) = make_uint4(sl8::pack_bf16x2(v[0], v[1]), sl8::pack_bf16x2(v[2], v[3]),
                                                  sl8::pack_bf16x2(v[4], v[5]), sl8::pack_bf16x2(v[6], v[7]));
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (32 * i < left) {
                if constexpr (sizeof(T) == 4) p[32 * i] = v[i];
                else p[32 * i] = __float2bfloat16_rn(v[i]);
            }
    }
}
template <bool VEC>
__device__ __forceinline__ void times_gamma(float (&v)[8], const float* gamma, int left) {      // gamma: shared memory
    if constexpr (VEC) {
        const float4 lo = reinterpret_cast<const float4*>(gamma)[0], hi = reinterpret_cast<const float4*>(gamma)[1];
        v[0] *= lo.x; v[1] *= lo.y; v[2] *= lo.z; v[3] *= lo.w;
        v[4] *= hi.x; v[5] *= hi.y; v[6] *= hi.z; v[7] *= hi.w;
    } else {
        if (left > 224) {
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] *= gamma[32 * i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (32 * i < left) v[i] *= gamma[32 * i];
        }
    }
}

// A row's codes are round(v * k), v = h * gamma (times rstd first where `small`).
struct Scaling {
    float rstd, scale, k;
    float rest;           // what rounding took from k (e4m3 codes of bf16 rows)
    bool small;
};
// A bf16 row as it is: its quotients v * 127 / max and v * 448 / max are often exactly half way between two codes (half of the largest is 63.5 steps of
// int8 in every row), and a factor that was rounded down or up would decide each of these for its whole row.
template <typename T, bool NORM>
constexpr bool kExact = !NORM && sizeof(T) == 2;

// v * k + 1.5 * 2^23, one rounding, leaves round-to-nearest-even(v * k) in the low byte (|v * k| < 127.5).
__device__ __forceinline__ uint32_t int8_of(float v, float k) { return __float_as_uint(fmaf(v, k, 12582912.0f)); }
__device__ __forceinline__ uint32_t int8x4(const float* v, float k) {
    return __byte_perm(__byte_perm(int8_of(v[0], k), int8_of(v[1], k), 0x0040), __byte_perm(int8_of(v[2], k), int8_of(v[3], k), 0x0040), 0x5410);
}
// EXACT: v * (k + rest), rounded once to fp32, is half way between two e4m3 codes (five bits) only where the quotient of the bf16 numbers is: any other
// quotient is at least 2^-13 of such a number away from it.  Two of them in two packed instructions, as many as v * k takes; volatile, or they are
// worked out for int8 codes too (46 656 x 4 304 int8 99 us, 93 so).
template <bool EXACT>
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi, const Scaling& s) {
    if constexpr (!EXACT) return sl8::pack_e4m3x2(lo * s.k, hi * s.k);
    uint32_t r;
    asm volatile(
        "{\n\t.reg .b64 v, k, e;\n\t.reg .b32 a, b;\n\t.reg .b16 c;\n\t"
        "mov.b64 v, {%1, %2};\n\tmov.b64 k, {%3, %3};\n\tmov.b64 e, {%4, %4};\n\t"
        "mul.rn.f32x2 e, v, e;\n\tfma.rn.f32x2 v, v, k, e;\n\tmov.b64 {a, b}, v;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 c, b, a;\n\tcvt.u32.u16 %0, c;\n\t}"
        : "=r"(r)
        : "f"(lo), "f"(hi), "f"(s.k), "f"(s.rest));
    return r;
}
template <bool EXACT>
__device__ __forceinline__ uint32_t e4m3x4(const float* v, const Scaling& s) {
    return e4m3x2<EXACT>(v[0], v[1], s) | (e4m3x2<EXACT>(v[2], v[3], s) << 16);
}
template <bool VEC, bool EXACT>
__device__ __forceinline__ void put_codes(uint8_t* p, const float (&v)[8], const Scaling& s, bool int8, int left) {
    const float k = s.k;
    if constexpr (VEC) {
        *reinterpret_cast<uint2*>(p) = int8 ? make_uint2(int8x4(v, k), int8x4(v + 4, k)) : make_uint2(e4m3x4<EXACT>(v, s), e4m3x4<EXACT>(v + 4, s));
    } else {
        uint32_t code[8];
        if (int8) {
#pragma unroll
            for (int i = 0; i < 8; i++) code[i] = int8_of(v[i], k);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                code[i] = e4m3x2<EXACT>(v[i], v[i + 1], s);
                code[i + 1] = code[i] >> 8;
            }
        }
        if (left > 224) {
#pragma unroll
            for (int i = 0; i < 8; i++) p[32 * i] = static_cast<uint8_t>(code[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (32 * i < left) p[32 * i] = static_cast<uint8_t>(code[i]);
        }
    }
}

// The largest of m and eight magnitudes; a NaN among them is the largest.
__device__ __forceinline__ float largest_of(float m, const float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(m), "f"(v[i]), "f"(v[i + 1]));
    return m;
}

struct Stats {
    float squares;        // sum of h^2
    float largest;        // largest |h * gamma|
};
template <bool NORM>
__device__ __forceinline__ Stats reduce_warp(Stats s) {
    if constexpr (NORM) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s.squares += __shfl_xor_sync(0xffffffffu, s.squares, o);
    }
    s.largest = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(s.largest)));     // (as integers: ordered like the numbers, NaN above infinity)
    return s;
}
// Over the threads of a block; `turn` counts the calls (they use two sets of partial results in turn, so one barrier does).
template <bool NORM>
__device__ __forceinline__ Stats reduce_block(Stats s, int turn) {
    __shared__ Stats part[2][32];
    s = reduce_warp<NORM>(s);
    const int lane = threadIdx.x & 31;
    if (lane == 0) part[turn & 1][threadIdx.x >> 5] = s;
    __syncthreads();
    return reduce_warp<NORM>(lane < static_cast<int>(blockDim.x >> 5) ? part[turn & 1][lane] : Stats{0.0f, 0.0f});
}

constexpr float kInfinity = __builtin_huge_valf(), kSmallest = 1.17549435e-38f /* 2^-126 */, kLargest = 3.40282347e38f;

template <bool NORM, bool EXACT>
__device__ __forceinline__ Scaling scaling(const RowArgs& a, const Stats& s, float given) {
    Scaling r;
    r.rest = 0.0f;
    const float nan = __int_as_float(0x7FC00000);
    // a sum of squares that is no number (an infinity or NaN among the elements, or squares beyond fp32): nothing that comes out is one
    r.rstd = !NORM ? 1.0f : s.squares < kInfinity ? __frsqrt_rn(__fdiv_rn(s.squares, static_cast<float>(a.cols)) + a.eps) : nan;
    r.small = false;
    if (!a.row_scales) {
        r.scale = 0.0f;
        r.k = __fdiv_rn(r.rstd, given);
        if (r.k > kLargest) r.k = kLargest;                   // (zeros stay zeros, the rest saturates)
        return r;
    }
    // rounding is monotonic: the largest |v| times rstd is the largest |v * rstd|.  127 / largest |v| takes rstd and the scale's rounding
    // out of the codes.
    const float top = a.int8 ? 127.0f : 448.0f, v = s.largest, y = v * r.rstd;
    if (y == 0.0f) {
        r.scale = 1.0f;
        r.k = 0.0f;
    } else if (y < kInfinity) {
        r.scale = __fdiv_rn(y, top);
        r.k = __fdiv_rn(top, v);
        if constexpr (EXACT) {
            // int8: a factor a little above 127 / max.  Of the quotients half way between two whole numbers it decides v = max / 2, and that belongs up, to 64;
            // any other, 254 v an odd multiple of max, has 127 divide max: mantissa 254, 127 / max exact and left as it is.
            // e4m3: one a little below 448 / max, and what is missing (above zero: a negative zero stays one).
            // (Divisions that round up or down: 46 656 x 4 304 int8 5 % more.)
            const bool above = a.int8 && (__float_as_int(v) & 0x7FFFFF) != 0x7E0000;
            r.k = __int_as_float(__float_as_int(r.k) + (a.int8 ? above : -1));
            r.rest = fmaf(-r.k, v, top) * (r.k * (1.0f / 448.0f));
        }
        if (r.scale < kSmallest || r.k > kLargest) {
            r.small = true;
            r.scale = fmaxf(r.scale, kSmallest);
            r.k = __frcp_rn(r.scale);
            r.rest = 0.0f;
        }
    } else {
        r.scale = r.k = nan;
    }
    return r;
}

// A row by the threads of a block (or, WARP, of a warp), CH times eight elements each: read once and held in registers, everything
// asked for before the first of it is used; statistics in fp32, four partial sums a thread.  For one wave of rows: bound by one trip
// to memory and the launch (one row of 1 152 bf16 with a residual 1.7 us, 8 rows of 4 304 1.5; 5 003 x 1 152 by warps 5.4).  Gamma
// comes through shared memory while the first row is on its way: kept in registers it costs a third of the warps (fp32 46 656 x 1 152
// 80 us, 65 so).
constexpr int kWarpRowThreads = 128;
template <typename T, bool NORM, bool VEC, int CH, bool WARP>
__global__ void __launch_bounds__(WARP ? kWarpRowThreads : CH == 1 ? 1024 : 512) row_kernel(const RowArgs a) {
    const int lane = threadIdx.x & 31;
    const int c0 = (WARP ? 0 : (threadIdx.x >> 5) * 256) + (VEC ? 8 * lane : lane), c_step = WARP ? 256 : 8 * blockDim.x;
    const auto column = [&](int j) { return c0 + c_step * j; };              // the first of the eight elements
    constexpr int ROWS = WARP ? kWarpRowThreads / 32 : 1;                    // of the block at a time
    sl8::pdl_wait();
    sl8::pdl_release();
    const float given = a.scale ? sl8::ld_f32(a.scale) : 1.0f;
    extern __shared__ __align__(16) float row_gamma[];                       // the block's copy: read again for every row
    if (NORM && a.gamma) {
        constexpr int PER = VEC ? 4 : 1;
        for (int c = PER * threadIdx.x; c < a.cols; c += PER * blockDim.x)
            asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(sl8::smem_u32(row_gamma + c)), "l"(a.gamma + c), "n"(4 * PER) : "memory");
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    int turn = 0;
    for (long long r0 = static_cast<long long>(blockIdx.x) * ROWS; r0 < a.rows; r0 += static_cast<long long>(gridDim.x) * ROWS, turn++) {
        const long long r = r0 + (WARP ? threadIdx.x >> 5 : 0);
        const bool live = !WARP || r < a.rows;                               // this warp has a row
        const T* const x = static_cast<const T*>(a.x) + r * a.ld;
        float v[CH][8];
        Stats s = {0.0f, 0.0f};
        if constexpr (NORM) {
            Eight<T> e[CH], f[CH];
#pragma unroll
            for (int j = 0; j < CH; j++)
                if (live && column(j) < a.cols) fetch<VEC>(e[j], x + column(j), a.cols - column(j));
            if (live && a.residual) {
                const T* const res = static_cast<const T*>(a.residual) + r * a.ld_res;
#pragma unroll
                for (int j = 0; j < CH; j++)
                    if (column(j) < a.cols) fetch<VEC>(f[j], res + column(j), a.cols - column(j));
            }
            if (turn == 0 && a.gamma) {       // (with the first row's elements on their way)
                asm volatile("cp.async.wait_all;" ::: "memory");
                __syncthreads();
            }
            if (!live) continue;
            float squares[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < CH; j++)
                if (column(j) < a.cols) {
#pragma unroll
                    for (int i = 0; i < 8; i++) v[j][i] = value(e[j], i);
                    if (a.residual) {
#pragma unroll
                        for (int i = 0; i < 8; i++) v[j][i] += value(f[j], i);
                        put_sum<VEC>(static_cast<T*>(a.sum) + r * a.ld_sum + column(j), v[j], a.cols - column(j));
                    }
#pragma unroll
                    for (int i = 0; i < 8; i++) squares[i & 3] = fmaf(v[j][i], v[j][i], squares[i & 3]);
                    if (a.gamma) times_gamma<VEC>(v[j], row_gamma + column(j), a.cols - column(j));
                    s.largest = largest_of(s.largest, v[j]);
                }
            s.squares = (squares[0] + squares[1]) + (squares[2] + squares[3]);
        } else {
            if (!live) continue;
            Eight<T> e[CH];
#pragma unroll
            for (int j = 0; j < CH; j++)
                if (column(j) < a.cols) fetch<VEC>(e[j], x + column(j), a.cols - column(j));
#pragma unroll
            for (int j = 0; j < CH; j++)
                if (column(j) < a.cols) {
#pragma unroll
                    for (int i = 0; i < 8; i++) v[j][i] = value(e[j], i);
                    s.largest = largest_of(s.largest, v[j]);
                }
        }
        const Scaling k = scaling<NORM, kExact<T, NORM>>(a, WARP ? reduce_warp<NORM>(s) : reduce_block<NORM>(s, turn), given);
        uint8_t* const out = a.out + r * a.ld_out;
#pragma unroll
        for (int j = 0; j < CH; j++)
            if (column(j) < a.cols) {
                if (k.small) {
#pragma unroll
                    for (int i = 0; i < 8; i++) v[j][i] *= k.rstd;
                }
                put_codes<VEC, kExact<T, NORM>>(out + column(j), v[j], k, a.int8 != 0, a.cols - column(j));
            }
        if (a.row_scales && (WARP ? lane : static_cast<int>(threadIdx.x)) == 0) a.row_scales[r] = k.scale;
    }
}

// Rows of up to 256 elements (heads, groups), many: LANES lanes to a row, eight elements a lane; its gamma stays in registers.  Bound by the
// bytes, and by what a row costs besides them (its reductions and divisions): bf16 -> int8 500 000 x 64 23 us (a warp to a row, ring 81), x 128
// 44 (81); norm with a residual 47 (167) and 91 (167), two rows of a lane at a time (one 53 and 104, four 50 and 94; without the
// norm one 23, two 25, four 27).  200 000 x 100 bf16, element by element, 30 (53).
constexpr int kNarrowThreads = 256;
__host__ __device__ constexpr int narrow_rows(bool norm, bool vec) { return norm && vec ? 2 : 1; }      // of a lane at a time
template <typename T, bool NORM, bool VEC, int LANES>
__global__ void __launch_bounds__(kNarrowThreads, !NORM && VEC ? 6 : NORM && sizeof(T) == 4 ? 3 : 4) narrow_row_kernel(const RowArgs a) {
    constexpr int U = narrow_rows(NORM, VEC), PER_WARP = 32 / LANES, STEP = VEC ? 1 : LANES;
    const int lane = threadIdx.x & 31, l = lane % LANES, c0 = VEC ? 8 * l : l;
    const int left = a.cols - c0;                                            // elements from this lane's first on
    sl8::pdl_wait();
    sl8::pdl_release();
    const float given = a.scale ? sl8::ld_f32(a.scale) : 1.0f;
    float g[8];
#pragma unroll
    for (int i = 0; i < 8; i++) g[i] = NORM && a.gamma && STEP * i < left ? sl8::ld_f32(a.gamma + c0 + STEP * i) : 1.0f;
    const long long warps = static_cast<long long>(gridDim.x) * (kNarrowThreads / 32);
    for (long long base = (blockIdx.x * static_cast<long long>(kNarrowThreads / 32) + (threadIdx.x >> 5)) * (PER_WARP * U); base < a.rows; base += warps * (PER_WARP * U)) {
        const long long first = base + lane / LANES;                         // this lane's rows: first, first + PER_WARP, ...
        const auto live = [&](int u) { return left > 0 && first + u * PER_WARP < a.rows; };
        const auto row = [&](const void* p, long long ld, int u) { return static_cast<const T*>(p) + (first + u * PER_WARP) * ld + c0; };
        const auto take = [&](Eight<T>& e, const T* p) {
            if constexpr (VEC) {
                fetch<true>(e, p, left);
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const T* const at = p + STEP * min(i, (left - 1) / STEP);         // (the last one in the place of those beyond)
                    uint32_t b;
                    if constexpr (sizeof(T) == 4) b = __float_as_uint(sl8::ld_f32(at));
                    else b = ld_u16(at);
                    if (STEP * i >= left) b = 0u;
                    if constexpr (sizeof(T) == 4) e.w[i] = b;
                    else if (i & 1) e.w[i / 2] |= b << 16;
                    else e.w[i / 2] = b;
                }
            }
        };
        Eight<T> e[U], f[U];
#pragma unroll
        for (int u = 0; u < U; u++)
            if (live(u)) take(e[u], row(a.x, a.ld, u));
        if (NORM && a.residual) {
#pragma unroll
            for (int u = 0; u < U; u++)
                if (live(u)) take(f[u], row(a.residual, a.ld_res, u));
        }
        float v[U][8];
        Stats s[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            s[u] = Stats{0.0f, 0.0f};
            if (!live(u)) continue;
#pragma unroll
            for (int i = 0; i < 8; i++) v[u][i] = value(e[u], i);
            if constexpr (NORM) {
                if (a.residual) {
#pragma unroll
                    for (int i = 0; i < 8; i++) v[u][i] += value(f[u], i);
                    T* const sum = static_cast<T*>(a.sum) + (first + u * PER_WARP) * a.ld_sum + c0;
                    if constexpr (VEC) {
                        put_sum<true>(sum, v[u], left);
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; i++)
                            if (STEP * i < left) {
                                if constexpr (sizeof(T) == 4) sum[STEP * i] = v[u][i];
                                else sum[STEP * i] = __float2bfloat16_rn(v[u][i]);
                            }
                    }
                }
                float odd = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    s[u].squares = fmaf(v[u][i], v[u][i], s[u].squares);
                    odd = fmaf(v[u][i + 1], v[u][i + 1], odd);
                }
                s[u].squares += odd;
#pragma unroll
                for (int i = 0; i < 8; i++) v[u][i] *= g[i];
            }
            s[u].largest = largest_of(0.0f, v[u]);
        }
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1)
#pragma unroll
            for (int u = 0; u < U; u++) {
                if constexpr (NORM) s[u].squares += __shfl_xor_sync(0xffffffffu, s[u].squares, o);
                s[u].largest = __uint_as_float(max(__float_as_uint(s[u].largest), __shfl_xor_sync(0xffffffffu, __float_as_uint(s[u].largest), o)));
            }
        // every lane knows the sums of its rows: of two rows, one lane in two works out one of them, and the others ask it
        Stats one = s[0];
        if (U == 2 && (l & 1)) one = s[U - 1];
        const Scaling of_one = scaling<NORM, kExact<T, NORM>>(a, one, given);
#pragma unroll
        for (int u = 0; u < U; u++) {
            Scaling k = of_one;
            if constexpr (U == 2) {
                const int from = lane / LANES * LANES + u;
                k.k = __shfl_sync(0xffffffffu, of_one.k, from);
                k.scale = __shfl_sync(0xffffffffu, of_one.scale, from);
                k.rstd = __shfl_sync(0xffffffffu, of_one.rstd, from);
                k.small = __shfl_sync(0xffffffffu, static_cast<int>(of_one.small), from) != 0;
            }
            if (!live(u)) continue;
            if (k.small) {
#pragma unroll
                for (int i = 0; i < 8; i++) v[u][i] *= k.rstd;
            }
            uint8_t* const out = a.out + (first + u * PER_WARP) * a.ld_out + c0;
            if constexpr (VEC) {
                put_codes<true, kExact<T, NORM>>(out, v[u], k, a.int8 != 0, left);
            } else {
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    const uint32_t two = a.int8 ? __byte_perm(int8_of(v[u][i], k.k), int8_of(v[u][i + 1], k.k), 0x0040) : e4m3x2<kExact<T, NORM>>(v[u][i], v[u][i + 1], k);
                    if (STEP * i < left) out[STEP * i] = static_cast<uint8_t>(two);
                    if (STEP * (i + 1) < left) out[STEP * (i + 1)] = static_cast<uint8_t>(two >> 8);
                }
            }
            if (a.row_scales && l == 0) a.row_scales[first + u * PER_WARP] = k.scale;
        }
    }
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
template <typename T>
__device__ __forceinline__ void shared_eight(Eight<T>& e, const T* p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; i++) {
        const uint4 q = *reinterpret_cast<const uint4*>(p + i * (16 / (int)sizeof(T)));
        e.w[4 * i] = q.x; e.w[4 * i + 1] = q.y; e.w[4 * i + 2] = q.z; e.w[4 * i + 3] = q.w;
    }
}
template <bool VEC, typename T>
__device__ __forceinline__ void shared_values(float (&v)[8], const T* p, int left) {
    if constexpr (VEC) {
        Eight<T> e;
        shared_eight(e, p);
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = value(e, i);
    } else {
        if (left > 224) {
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = static_cast<float>(p[32 * i]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = 32 * i < left ? static_cast<float>(p[32 * i]) : 0.0f;
        }
    }
}

// The same for many rows: each block (or, WARP, warp) has a ring of two slots in shared memory and asks for a row, one bulk copy for x and
// one for the residual, as soon as the one two before it has been read, so that there is always a row on its way and the registers
// hold one only.  Bound by the bytes: 46 656 x 4 304 bf16 -> int8 93 us, the copy rate of this memory (rows in registers 115);
// RMS norm of 16 384 x 4 096 with a residual 78 us, 6.0 TB/s (84); 46 656 x 1 152 fp32 -> e4m3 49 us, 5.5 TB/s (65).  Three slots
// were slower nearly everywhere (16 384 x 4 096 81 us: fewer blocks fit).
// Rows on any address: the copy takes the 16-byte granules that the row touches, and lanes read consecutive elements from there.  5 003 x 4 305
// bf16 18.0 us, 3.6 TB/s (from memory, lane by lane, 52: a warp's loads of 64 bytes do not keep enough in flight); the codes go out byte by byte.
constexpr int kSlots = 2;
__host__ __device__ constexpr int gamma_bytes(bool given, int cols) { return given ? (cols + 255) / 256 * 1024 : 0; }
template <typename T, bool NORM, bool VEC, int CH, bool WARP>
__global__ void __launch_bounds__(WARP ? kWarpRowThreads : 512) row_stream_kernel(const RowArgs a, int span) {
    constexpr int GROUPS = WARP ? kWarpRowThreads / 32 : 1;
    extern __shared__ __align__(128) uint8_t stream_smem[];
    __shared__ __align__(8) uint64_t bars[GROUPS * kSlots];
    __shared__ volatile uint32_t abort_flag;
    const int lane = threadIdx.x & 31, group = WARP ? threadIdx.x >> 5 : 0;
    const bool lead = WARP ? lane == 0 : threadIdx.x == 0;
    const int c0 = (WARP ? 0 : (threadIdx.x >> 5) * 256) + (VEC ? 8 * lane : lane), c_step = WARP ? 256 : 8 * blockDim.x;
    const auto column = [&](int j) { return c0 + c_step * j; };
    const bool gamma = NORM && a.gamma, residual = NORM && a.residual;
    float* const g = reinterpret_cast<float*>(stream_smem);
    const int slot_bytes = residual ? 2 * span : span;
    uint8_t* const slots = stream_smem + gamma_bytes(gamma, a.cols) + group * kSlots * slot_bytes;
    const uint32_t bar0 = sl8::smem_u32(bars + group * kSlots);
    sl8::WaitCtx wc;
    wc.abort_flag = &abort_flag;
    wc.peer_abort = 0u;
    wc.status = a.status;
    wc.budget_ns = static_cast<unsigned long long>(a.wait_budget_us) * 1000ull;
    wc.tile = 0;
    if (lead) {
        for (int s = 0; s < kSlots; s++) sl8::mbar_init(bar0 + 8 * s, 1);
        sl8::fence_mbar_init();
        if (group == 0) abort_flag = 0u;
    }
    sl8::pdl_wait();
    sl8::pdl_release();
    const float given = a.scale ? sl8::ld_f32(a.scale) : 1.0f;
    const long long stride = static_cast<long long>(gridDim.x) * GROUPS;
    // Bytes of a row from the 16-byte boundary at or below its start to the one at or above its end.  What sticks out belongs to the rows
    // beside it (a row has at least 16 bytes); of the first and the last row it may not belong to the caller, so these are read element by element.
    const auto apart = [&](long long r) { return !VEC && (r == 0 || r == a.rows - 1); };
    const auto issue = [&](int s, long long r) {
        if (r >= a.rows || apart(r) || !lead) return;
        const uint32_t dst = sl8::smem_u32(slots + s * slot_bytes), bar = bar0 + 8 * s;
        const auto one = [&](const void* p, long long ld, uint32_t to, bool copy) {
            const uintptr_t from = reinterpret_cast<uintptr_t>(p) + r * ld * sizeof(T), start = from & ~uintptr_t{15};
            const uint32_t bytes = static_cast<uint32_t>((from + a.cols * sizeof(T) + 15) / 16 * 16 - start);
            if (copy) bulk_load(to, reinterpret_cast<const void*>(start), bytes, bar);
            return bytes;
        };
        const uint32_t total = one(a.x, a.ld, dst, false) + (residual ? one(a.residual, a.ld_res, dst + span, false) : 0u);
        if (!VEC) sl8::fence_proxy_async_smem();       // (rows that are read element by element are written to their slot)
        sl8::mbar_arrive_expect_tx(bar, total);
        if (!(a.drop && r == 1)) one(a.x, a.ld, dst, true);
        if (residual) one(a.residual, a.ld_res, dst + span, true);
    };
    long long r = blockIdx.x * static_cast<long long>(GROUPS) + group;
    for (int s = 0; s < kSlots; s++) issue(s, r + s * stride);
    if (gamma) {
        constexpr int PER = VEC ? 4 : 1;
        for (int c = PER * threadIdx.x; c < a.cols; c += PER * blockDim.x) {
            // VEC: the two halves of a lane's eight 128 elements apart, so that the lanes' reads meet no bank twice
            const int to = VEC ? (c & ~255) + ((c & 4) ? 128 : 0) + (c & 255) / 8 * 4 : c;
            asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(sl8::smem_u32(g + to)), "l"(a.gamma + c), "n"(4 * PER) : "memory");
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    }
    __syncthreads();
    uint32_t phases = 0u;
    for (int turn = 0, s = 0; r < a.rows; r += stride, turn++, s = s + 1 == kSlots ? 0 : s + 1) {
        uint8_t* const slot = slots + s * slot_bytes;
        const auto place = [&](const void* p, long long ld, uint8_t* at) {        // where the row's elements lie in the slot
            return reinterpret_cast<T*>(at + (VEC ? 0 : (reinterpret_cast<uintptr_t>(p) + r * ld * sizeof(T)) & 15));
        };
        T* const x = place(a.x, a.ld, slot);
        T* const res = place(a.residual, a.ld_res, slot + span);
        bool ok = true;
        if (apart(r)) {
            const int first = WARP ? lane : threadIdx.x, step = WARP ? 32 : blockDim.x;
            for (int c = first; c < a.cols; c += step) {
                x[c] = static_cast<const T*>(a.x)[r * a.ld + c];
                if (residual) res[c] = static_cast<const T*>(a.residual)[r * a.ld_res + c];
            }
            if (WARP) __syncwarp();
            else __syncthreads();
        } else {
            wc.tile = static_cast<uint32_t>(r);
            ok = sl8::wait_bar<true>(bar0 + 8 * s, (phases >> s) & 1u, wc, sl8::ST_ROW_WAIT, s);
            phases ^= 1u << s;
        }
        // a row that has not come is not touched (its sum may go where x or the residual is): all of its threads know before the first writes
        if (WARP ? !__all_sync(0xffffffffu, ok) : residual && !__syncthreads_and(ok)) break;
        float v[CH][8];
        Stats st = {0.0f, 0.0f};
        float squares[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < CH; j++)
            if (column(j) < a.cols) {
                const int left = a.cols - column(j);
                shared_values<VEC>(v[j], x + column(j), left);
                if constexpr (NORM) {
                    if (residual) {
                        float f[8];
                        shared_values<VEC>(f, res + column(j), left);
#pragma unroll
                        for (int i = 0; i < 8; i++) v[j][i] += f[i];
                        put_sum<VEC>(static_cast<T*>(a.sum) + r * a.ld_sum + column(j), v[j], left);
                    }
#pragma unroll
                    for (int i = 0; i < 8; i++) squares[i & 3] = fmaf(v[j][i], v[j][i], squares[i & 3]);
                    if (gamma) {
                        if constexpr (VEC) {
                            const float* const at = g + (column(j) & ~255) + 4 * lane;
                            const float4 lo = *reinterpret_cast<const float4*>(at), hi = *reinterpret_cast<const float4*>(at + 128);
                            v[j][0] *= lo.x; v[j][1] *= lo.y; v[j][2] *= lo.z; v[j][3] *= lo.w;
                            v[j][4] *= hi.x; v[j][5] *= hi.y; v[j][6] *= hi.z; v[j][7] *= hi.w;
                        } else {
                            times_gamma<VEC>(v[j], g + column(j), left);
                        }
                    }
                }
                st.largest = largest_of(st.largest, v[j]);
            }
        st.squares = (squares[0] + squares[1]) + (squares[2] + squares[3]);
        st = WARP ? reduce_warp<NORM>(st) : reduce_block<NORM>(st, turn);
        if (WARP) __syncwarp();
        else if (abort_flag) break;              // (set ahead of the barrier by whoever gave up: seen by all)
        issue(s, r + kSlots * stride);
        const Scaling k = scaling<NORM, kExact<T, NORM>>(a, st, given);
        uint8_t* const out = a.out + r * a.ld_out;
#pragma unroll
        for (int j = 0; j < CH; j++)
            if (column(j) < a.cols) {
                if (k.small) {
#pragma unroll
                    for (int i = 0; i < 8; i++) v[j][i] *= k.rstd;
                }
                put_codes<VEC, kExact<T, NORM>>(out + column(j), v[j], k, a.int8 != 0, a.cols - column(j));
            }
        if (a.row_scales && lead) a.row_scales[r] = k.scale;
    }
    if (abort_flag) {          // copies in flight land before their memory is released
        const unsigned long long t0 = sl8::globaltimer_ns();
        while (sl8::globaltimer_ns() - t0 < 200000ull) {
        }
    }
}

// Rows too long for the registers of a block, or for its ring: read twice, statistics first.  The sum is written the second time only, because it may
// lie where the second reading still has to find x or the residual.
constexpr int kLongThreads = 512;
template <typename T, bool NORM, bool VEC>
__global__ void __launch_bounds__(kLongThreads) long_row_kernel(const RowArgs a) {
    const int first = VEC ? 8 * threadIdx.x : (threadIdx.x >> 5) * 256 + (threadIdx.x & 31);
    sl8::pdl_wait();
    sl8::pdl_release();
    const float given = a.scale ? sl8::ld_f32(a.scale) : 1.0f;
    int turn = 0;
    for (long long r = blockIdx.x; r < a.rows; r += gridDim.x, turn++) {
        const T* const x = static_cast<const T*>(a.x) + r * a.ld;
        // h of the group at column c
        const auto load = [&](int c, float (&v)[8], bool write) {
            Eight<T> e, f;
            fetch<VEC>(e, x + c, a.cols - c);
            if (NORM && a.residual) fetch<VEC>(f, static_cast<const T*>(a.residual) + r * a.ld_res + c, a.cols - c);
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = value(e, i);
            if (NORM && a.residual) {
#pragma unroll
                for (int i = 0; i < 8; i++) v[i] += value(f, i);
                if (write) put_sum<VEC>(static_cast<T*>(a.sum) + r * a.ld_sum + c, v, a.cols - c);
            }
        };
        const auto scaled = [&](int c, float (&v)[8]) {
            if (NORM && a.gamma) {
                Eight<float> g;
                fetch<VEC>(g, a.gamma + c, a.cols - c);
#pragma unroll
                for (int i = 0; i < 8; i++) v[i] *= value(g, i);
            }
        };
        Stats s = {0.0f, 0.0f};
        float squares[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int c = first; c < a.cols; c += 8 * kLongThreads) {
            float v[8];
            load(c, v, false);
            if constexpr (NORM) {
#pragma unroll
                for (int i = 0; i < 8; i++) squares[i & 3] = fmaf(v[i], v[i], squares[i & 3]);
                scaled(c, v);
            }
            s.largest = largest_of(s.largest, v);
        }
        s.squares = (squares[0] + squares[1]) + (squares[2] + squares[3]);
        const Scaling k = scaling<NORM, kExact<T, NORM>>(a, reduce_block<NORM>(s, turn), given);
        for (int c = first; c < a.cols; c += 8 * kLongThreads) {
            float v[8];
            load(c, v, true);
            scaled(c, v);
            if (k.small) {
#pragma unroll
                for (int i = 0; i < 8; i++) v[i] *= k.rstd;
            }
            put_codes<VEC, kExact<T, NORM>>(a.out + r * a.ld_out + c, v, k, a.int8 != 0, a.cols - c);
        }
        if (a.row_scales && threadIdx.x == 0) a.row_scales[r] = k.scale;
    }
}

// ---- which kernel, on how many blocks
constexpr size_t kRingBytes = 227 * 1024 - 1024;       // shared memory of a block, less what the kernel declares itself
constexpr size_t kDirectBytes = 12288 * sizeof(float); // gamma of the widest rows of row_kernel
// Leave to launch with `bytes` of shared memory (48 KiB need none, what the kernel declares itself included).  It belongs to the kernel on the
// device, which every thread and handle shares: each asks for the same, the most that any call can need, so none takes another's away.
template <typename Kernel>
cudaError_t allow_shared(Kernel kernel, size_t bytes, size_t most) {
    return bytes > 40 * 1024 ? cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(most)) : cudaSuccess;
}

template <typename T, bool NORM, bool VEC>
cudaError_t launch_long(int sm_count, cudaStream_t s, const RowArgs& a) {
    const long long cap = static_cast<long long>(sm_count) * 8;
    return sl8_launch_chained(long_row_kernel<T, NORM, VEC>, static_cast<unsigned>(a.rows < cap ? a.rows : cap), kLongThreads, 0, s, a);
}

template <typename T, bool NORM, bool VEC, int CH, bool WARP>
cudaError_t direct(int sm_count, cudaStream_t s, const RowArgs& a) {
    const auto kernel = row_kernel<T, NORM, VEC, CH, WARP>;
    const size_t bytes = NORM && a.gamma ? sizeof(float) * a.cols : 0;
    const cudaError_t e = allow_shared(kernel, bytes, kDirectBytes);
    if (e != cudaSuccess) return e;
    constexpr int ROWS = WARP ? kWarpRowThreads / 32 : 1;
    const int threads = WARP ? kWarpRowThreads : ((a.cols + 7) / 8 + CH * 32 - 1) / (CH * 32) * 32;
    const long long want = (a.rows + ROWS - 1) / ROWS, cap = static_cast<long long>(sm_count) * (WARP ? 16 : 8);
    return sl8_launch_chained(kernel, static_cast<unsigned>(want < cap ? want : cap), threads, bytes, s, a);
}

template <typename T, bool NORM, bool VEC, int CH, bool WARP>
cudaError_t stream_rows(int sm_count, cudaStream_t s, const RowArgs& a) {
    const auto kernel = row_stream_kernel<T, NORM, VEC, CH, WARP>;
    static const int regs = [&] {                       // of the kernel, looked up once
        cudaFuncAttributes fa = {};
        return cudaFuncGetAttributes(&fa, kernel) == cudaSuccess && fa.numRegs > 0 ? fa.numRegs : 64;
    }();
    constexpr int GROUPS = WARP ? kWarpRowThreads / 32 : 1;
    const int span = (a.cols * static_cast<int>(sizeof(T)) + 16 + 127) / 128 * 128;
    const size_t bytes = gamma_bytes(NORM && a.gamma, a.cols) + static_cast<size_t>(GROUPS) * kSlots * span * (a.residual ? 2 : 1);
    if (bytes > kRingBytes) return launch_long<T, NORM, VEC>(sm_count, s, a);
    const cudaError_t e = allow_shared(kernel, bytes, kRingBytes);
    if (e != cudaSuccess) return e;
    const int threads = WARP ? kWarpRowThreads : ((a.cols + 7) / 8 + CH * 32 - 1) / (CH * 32) * 32;
    // Blocks that are resident at once, and from some rows per block on several times as many: the SMs do not get through their rows
    // equally fast.  Each block brings gamma once, so that one with gamma takes more rows.
    const int by_regs = 65536 / ((regs + 7) / 8 * 8 * threads), by_bytes = static_cast<int>(228 * 1024 / (bytes + 2048)), by_warps = 2048 / threads;
    int resident = by_regs < by_bytes ? by_regs : by_bytes;
    if (by_warps < resident) resident = by_warps;
    if (resident < 1) resident = 1;
    const long long want = (a.rows + GROUPS - 1) / GROUPS, once = static_cast<long long>(sm_count) * resident;
    long long waves = want / once / (WARP ? 4 : NORM && a.gamma ? 16 : 8);
    waves = want <= 2 * once ? 2 : waves < 1 ? 1 : waves > 4 ? 4 : waves;
    return sl8_launch_chained(kernel, static_cast<unsigned>(want < once * waves ? want : once * waves), threads, bytes, s, a, span);
}

template <typename T, bool NORM, bool VEC, int LANES>
cudaError_t narrow(int sm_count, cudaStream_t s, const RowArgs& a) {
    constexpr int ROWS = kNarrowThreads / LANES * narrow_rows(NORM, VEC);
    const long long want = (a.rows + ROWS - 1) / ROWS, cap = static_cast<long long>(sm_count) * 16;
    return sl8_launch_chained(narrow_row_kernel<T, NORM, VEC, LANES>, static_cast<unsigned>(want < cap ? want : cap), kNarrowThreads, 0, s, a);
}

bool few_rows(int sm_count, const RowArgs& a) { return a.rows <= 10ll * sm_count; }

// Up to ten rows per SM: a block each, one trip to memory (1 500 x 4 304 bf16 -> int8 5.9 us, ring 6.7); with all eight elements of a
// thread's at once while 256 threads do (norm of one row of 1 152 1.74 us, 1.95 with three times eight), with three from there on (729 x 4 304
// 3.6 us, 5.4 with one).  Of up to 256 elements: several to a warp.  Up to forty rows per SM, where they are short: a warp each (norm of 5 003 x 1 152 10.3 us, ring 10.9).  Then the ring, by
// warps while rows are short, by blocks of three times eight elements a thread (100 000 x 512 57 us by warps, 64 by blocks; 20 000 x
// 2 048 50 either way; 46 656 x 4 304 two us less than with four, four less than with two), and rows on odd addresses from the tenth row per SM (norm of
// 5 003 x 1 155 15.5 us, in registers 30).
template <typename T, bool NORM, bool VEC>
cudaError_t launch_rows(int sm_count, cudaStream_t s, const RowArgs& a) {
    const bool few = few_rows(sm_count, a);
    if (!few && a.cols <= 256) return a.cols <= 64 ? narrow<T, NORM, VEC, 8>(sm_count, s, a) : a.cols <= 128 ? narrow<T, NORM, VEC, 16>(sm_count, s, a) : narrow<T, NORM, VEC, 32>(sm_count, s, a);
    if (few) {
        if (a.cols <= 2048) return direct<T, NORM, VEC, 1, false>(sm_count, s, a);
        if (a.cols <= 12288) return direct<T, NORM, VEC, 3, false>(sm_count, s, a);
    }
    if constexpr (VEC) {
        if (a.rows <= 40ll * sm_count && a.cols <= 1280)
            return a.cols <= 768 ? direct<T, NORM, true, 3, true>(sm_count, s, a) : direct<T, NORM, true, 5, true>(sm_count, s, a);
        if (a.cols > 768 && a.cols <= 1280) return stream_rows<T, NORM, true, 5, true>(sm_count, s, a);
    }
    if (a.cols <= 512) return stream_rows<T, NORM, VEC, 2, true>(sm_count, s, a);
    if (a.cols <= 768) return stream_rows<T, NORM, VEC, 3, true>(sm_count, s, a);
    if constexpr (!VEC)
        if (a.cols <= 2048) return stream_rows<T, NORM, false, 2, false>(sm_count, s, a);
    if (a.cols <= 12288) return stream_rows<T, NORM, VEC, 3, false>(sm_count, s, a);
    if (a.cols <= 16384) return stream_rows<T, NORM, VEC, 4, false>(sm_count, s, a);
    return launch_long<T, NORM, VEC>(sm_count, s, a);
}

// The kernels with a ring take rows by bulk copies, which are for memory of a GPU (asked only where one may be taken: 0.1 us on the host).
bool on_the_host(const void* p) {
    cudaPointerAttributes at = {};
    if (!p || cudaPointerGetAttributes(&at, p) != cudaSuccess) {
        (void)cudaGetLastError();
        return false;
    }
    return at.type == cudaMemoryTypeHost || at.type == cudaMemoryTypeUnregistered;
}

template <typename T, bool NORM>
int run_rows(sl8_handle_t h, const RowArgs& a, sl8_stream_t stream, const char* what) {
    Sl8DeviceGuard guard(h->device);
    if (!guard.ok) return sl8_fail(h, SL8_ERR_CUDA, "cudaSetDevice failed");
    if (!few_rows(h->sm_count, a) && a.cols > 256 && (on_the_host(a.x) || on_the_host(a.residual)))
        return sl8_fail(h, SL8_ERR_INVALID_VALUE, "x and residual must be device memory: host memory is not copied in bulk");
    constexpr int PER_16 = 16 / sizeof(T);
    // eight elements per access where every row allows it, element by element otherwise
    const bool vec = a.cols % 8 == 0 && sl8_aligned16(a.x) && a.ld % PER_16 == 0 && a.ld_out % 8 == 0 && (reinterpret_cast<uintptr_t>(a.out) & 7u) == 0 &&
                     (!a.gamma || sl8_aligned16(a.gamma)) &&
                     (!a.residual || (sl8_aligned16(a.residual) && a.ld_res % PER_16 == 0 && sl8_aligned16(a.sum) && a.ld_sum % PER_16 == 0));
    const cudaError_t e = vec ? launch_rows<T, NORM, true>(h->sm_count, static_cast<cudaStream_t>(stream), a)
                              : launch_rows<T, NORM, false>(h->sm_count, static_cast<cudaStream_t>(stream), a);
    return e == cudaSuccess ? SL8_OK : sl8_fail_cuda(h, e, what);
}

constexpr int kMostColumns = 1 << 30;       // columns are counted in steps of 32 bits
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
    if (cols > kMostColumns) return sl8_fail(h, SL8_ERR_UNSUPPORTED, "more than 2^30 columns");
    if (!element_aligned(x, dtype) || !float_aligned(row_scales)) return sl8_fail(h, SL8_ERR_ALIGNMENT, "x and row_scales must be aligned to their elements");
    RowArgs a = {};
    a.x = x; a.ld = ld;
    a.out = static_cast<uint8_t*>(out); a.ld_out = ld_out;
    a.row_scales = row_scales; a.rows = rows; a.cols = cols; a.int8 = code_type == SL8_CODE_INT8;
    a.status = h->d_status; a.wait_budget_us = h->wait_budget_us; a.drop = h->test_drop_b;
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
    if (cols > kMostColumns) return sl8_fail(h, SL8_ERR_UNSUPPORTED, "more than 2^30 columns");
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
    a.status = h->d_status; a.wait_budget_us = h->wait_budget_us; a.drop = h->test_drop_b;
    return dtype == SL8_DT_F32 ? run_rows<float, true>(h, a, stream, "rmsnorm kernel launch") : run_rows<bf16, true>(h, a, stream, "rmsnorm kernel launch");
}
