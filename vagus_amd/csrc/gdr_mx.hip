// Rows and weights to block-scaled numbers (gdr_mx.hpp): the kernels that write them.
#include "gdr_kernels.hpp"
#include "gdr_mx.hpp"

namespace vgdr {

namespace {

// Eight elements of a row from column c on, as fp32; zeros from column n on.
template <typename E>
__device__ __forceinline__ void load8(float (&v)[8], const E *row, int64_t c, int64_t n, bool vec) {
    if (vec && c + 8 <= n) {
        constexpr int VE = 16 / (int)sizeof(E);
        typedef E V __attribute__((ext_vector_type(VE)));
#pragma unroll
        for (int u = 0; u < 8 / VE; ++u) {
            const V x = *reinterpret_cast<const V *>(row + c + u * VE);
#pragma unroll
            for (int e = 0; e < VE; ++e) v[u * VE + e] = (float)x[e];
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = c + e < n ? (float)row[c + e] : 0.f;
}

// the largest |v| of a block whose four lanes hold eight elements each, as fp32 bits (a NaN's are larger than any)
__device__ __forceinline__ uint32_t block_amax(const float (&v)[8]) {
    uint32_t m = abs_bits(v[0]);
#pragma unroll
    for (int e = 1; e < 8; ++e) m = max(m, abs_bits(v[e]));
    m = max(m, (uint32_t)__shfl_xor((int)m, 1));
    return max(m, (uint32_t)__shfl_xor((int)m, 2));
}

// a lane's eight elements of a block and (first lane of it) its scale
__device__ __forceinline__ void store8(uint8_t *values, uint8_t *scales, int64_t at, const float (&v)[8]) {
    const int b = mx_scale<8>(block_amax(v));
    *reinterpret_cast<u32x2 *>(values + at) = u32x2{mx_pack8(v, b), mx_pack8(v + 4, b)};
    if (at % 32 == 0) scales[at / 32] = (uint8_t)b;
}

}  // namespace

// Rows x [R, K] (ldx apart) to 8 bits: b = 2^s the smallest with amax <= 464 b, v = rne(x / b), exact but for that one
// rounding.  A thread eight elements, four threads a block: 16-byte loads, 8-byte stores, whole
// lines of both per wave, and the block's largest in two exchanges between neighbours.  Bound by
// memory: 65,536 rows of 2048 in bf16 71.9 us, 407 MB at 5.7 TB/s.
template <typename E>
__global__ void __launch_bounds__(256) mx_rows_kernel(const E *__restrict__ x, int64_t ldx, uint8_t *values,
                                                      uint8_t *scales, int64_t rows, int64_t K, int64_t Kp, bool vec) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, per = Kp / 8, row = i / per;
    if (row >= rows) return;                                          // whole blocks: per is a multiple of 16
    const int64_t c = (i - row * per) * 8;
    float v[8];
    load8(v, x + row * ldx, c, K, vec);
    store8(values, scales, row * Kp + c, v);
}

// Weights w [n, K] (ldw apart) to 4 bits in the tiles' order: a wave a tile, lane 16 g + r one block, whose 16 bytes it
// stores at its own place (a wave's stores are one run of 1024 bytes).  Four waves take the four tiles whose
// scales share words.  Bound by memory: 8192 x 8192 in bf16 34 us, 170 MB at 5.0 TB/s (element by element 148).
template <typename E>
__global__ void __launch_bounds__(256) mx_weight_kernel(const E *__restrict__ w, int64_t ldw, uint8_t *values,
                                                        uint8_t *scales, int64_t n, int64_t K, int64_t C, int64_t tiles,
                                                        bool gated, bool vec) {
    const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int64_t C4 = (C + 3) / 4, t = unit / (4 * C4), c = unit - t * 4 * C4;   // c past C: a scale alone
    if (t >= tiles) return;
    const int lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
    const int64_t half = n / 2;
    const int64_t in = 16 * (gated ? t / 2 : t) + r;                  // the row within its half
    const bool live = in < (gated ? half : n) && c < C;
    const E *row = w + (gated ? (t & 1) * half + in : in) * ldw;
    float v[32];
    uint32_t amax = 0;
#pragma unroll
    for (int e = 0; e < 32; e += 8) load8(*reinterpret_cast<float(*)[8]>(v + e), row, 128 * c + 32 * g + e, live ? K : 0, vec);
#pragma unroll
    for (int e = 0; e < 32; ++e) amax = max(amax, abs_bits(v[e]));
    const int b = mx_scale<4>(amax);
    if (c < C) {
        const float inv = b == 255 ? 0.f : mx_inverse(b);
        u32x4 q;
#pragma unroll
        for (int i = 0; i < 4; ++i) {                                 // the conversion rounds to even and saturates
            uint32_t p = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0, v[8 * i] * inv, v[8 * i + 1] * inv, 1.f, 0);
            p = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(p, v[8 * i + 2] * inv, v[8 * i + 3] * inv, 1.f, 1);
            p = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(p, v[8 * i + 4] * inv, v[8 * i + 5] * inv, 1.f, 2);
            q[i] = b == 255 ? 0x77777777u
                            : __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(p, v[8 * i + 6] * inv, v[8 * i + 7] * inv, 1.f, 3);
        }
        *reinterpret_cast<u32x4 *>(values + ((t * C + c) * 64 + lane) * 16) = q;
    }
    scales[((t * C4 + c / 4) * 64 + lane) * 4 + c % 4] = (uint8_t)b;
}

// h = x + residual, y = h rsqrt(mean h^2 + eps) gamma, y to 8 bits; a workgroup a row, a thread U units of eight
// elements, in registers from the read to the rounding: every byte moves once.  y is formed in 64 bits and rounded once
// (round_to_odd), so that the bytes are those of the formula itself, whatever the order of the sum; a multiply and an
// add in 64 bits an element, and three multiplies, lie under the loads.  Bound by memory: 65,536 rows of
// 2048 in bf16 with the residual 182 us, 945 MB at 5.2 TB/s; one row 2.5 us, a launch and two dependent round trips.
template <typename E, int U>
__global__ void __launch_bounds__(256) mx_rms_norm_kernel(const E *x, const E *res, E *x_out, const E *__restrict__ gamma,
                                                          float eps, E *y, uint8_t *values, uint8_t *scales, int dim,
                                                          int Kp) {
    constexpr int VE = 16 / (int)sizeof(E), VN = 8 / VE;
    typedef E V __attribute__((ext_vector_type(VE)));
    __shared__ double part[4];
    const int tid = threadIdx.x, nu = dim / 8, np = Kp / 8;
    const int64_t base = (int64_t)blockIdx.x * dim;
    float h[U][8];
    double ss = 0.;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int i = tid + 256 * u;
        if (i < nu) {
#pragma unroll
            for (int q = 0; q < VN; ++q) {
                const int64_t at = base + 8 * (int64_t)i + q * VE;
                V hv = *reinterpret_cast<const V *>(x + at);
                if (res) {
                    const V rv = *reinterpret_cast<const V *>(res + at);
#pragma unroll
                    for (int e = 0; e < VE; ++e) hv[e] = (E)((float)hv[e] + (float)rv[e]);
                }
                if (x_out) *reinterpret_cast<V *>(x_out + at) = hv;
#pragma unroll
                for (int e = 0; e < VE; ++e) {
                    h[u][q * VE + e] = (float)hv[e];
                    ss += (double)h[u][q * VE + e] * h[u][q * VE + e];
                }
            }
        }
    }
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) ss += __shfl_xor(ss, m);
    if ((tid & 63) == 0) part[tid >> 6] = ss;
    __syncthreads();
    const double r = 1. / sqrt((part[0] + part[1] + part[2] + part[3]) / dim + (double)eps);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int i = tid + 256 * u;
        if (i < np) {
            float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            if (i < nu) {
#pragma unroll
                for (int q = 0; q < VN; ++q) {
                    const V gv = *reinterpret_cast<const V *>(gamma + 8 * i + q * VE);
                    V o;
#pragma unroll
                    for (int e = 0; e < VE; ++e) {
                        v[q * VE + e] = round_to_odd(h[u][q * VE + e] * r * (double)(float)gv[e]);
                        o[e] = (E)((float)(E)(h[u][q * VE + e] * (float)r) * (float)gv[e]);
                    }
                    if (y) *reinterpret_cast<V *>(y + base + 8 * (int64_t)i + q * VE) = o;
                }
            }
            store8(values, scales, (int64_t)blockIdx.x * Kp + 8 * i, v);
        }
    }
}

// Many rows of fp16 or fp32 (or of bf16 of a width that is no multiple of 128) as bf16 planes [P][R][Kp] whose sum they are.  A
// product of a plane's element with a 4-bit weight is exact in fp32, so the tiles need one form of 16-bit rows, whose K
// steps are two or three times as many.  65,536 rows of 2048 against 8192 columns, planes and product: bf16 1,730 us (no
// planes), fp16 3,390, fp32 5,320 (the library's fp32 product alone: 14,400 at its rate of 153 TFLOP/s).
template <typename E, int P>
__global__ void __launch_bounds__(256) mx_planes_kernel(const E *__restrict__ x, int64_t ldx, __bf16 *out, int64_t rows,
                                                        int64_t K, int64_t Kp, bool vec) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, per = Kp / 8, row = i / per;
    if (row >= rows) return;
    const int64_t c = (i - row * per) * 8;
    float v[8];
    load8(v, x + row * ldx, c, K, vec);
    bf16x8 o[P];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        __bf16 part[P];
        split(part, v[e]);
#pragma unroll
        for (int p = 0; p < P; ++p) o[p][e] = part[p];
    }
#pragma unroll
    for (int p = 0; p < P; ++p) *reinterpret_cast<bf16x8 *>(out + (p * rows + row) * Kp + c) = o[p];
}

namespace {

template <typename E>
hipError_t quantize_t(const MxQuantize &p, hipStream_t stream) {
    const E *x = reinterpret_cast<const E *>(p.x);
    const bool vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && p.ldx * (int64_t)sizeof(E) % 16 == 0;
    const int64_t Kp = (p.K + 127) / 128 * 128;
    if (p.kind == MX_ROWS || p.kind == MX_PLANES) {
        const dim3 grid((unsigned)((p.rows * (Kp / 8) + 255) / 256));
        if (p.kind == MX_ROWS)
            hipLaunchKernelGGL((mx_rows_kernel<E>), grid, dim3(256), 0, stream, x, p.ldx, p.values, p.scales, p.rows, p.K, Kp, vec);
        else
            hipLaunchKernelGGL((mx_planes_kernel<E, mx_planes<E>()>), grid, dim3(256), 0, stream, x, p.ldx,
                               reinterpret_cast<__bf16 *>(p.values), p.rows, p.K, Kp, vec);
        return hipGetLastError();
    }
    const int64_t C = Kp / 128, tiles = p.gated ? 2 * ((p.rows / 2 + 15) / 16) : (p.rows + 15) / 16;
    hipLaunchKernelGGL((mx_weight_kernel<E>), dim3((unsigned)(tiles * ((C + 3) / 4))), dim3(256), 0, stream, x, p.ldx, p.values,
                       p.scales, p.rows, p.K, C, tiles, p.gated, vec);
    return hipGetLastError();
}

template <typename E>
hipError_t norm_t(const MxNorm &p, hipStream_t stream) {
    const E *x = reinterpret_cast<const E *>(p.x), *r = reinterpret_cast<const E *>(p.residual),
            *g = reinterpret_cast<const E *>(p.gamma);
    E *xo = reinterpret_cast<E *>(p.x_out), *y = reinterpret_cast<E *>(p.y);
    const int Kp = (p.dim + 127) / 128 * 128, units = Kp / 8;
    const dim3 grid((unsigned)p.rows);
    auto go = [&](auto u) {
        hipLaunchKernelGGL((mx_rms_norm_kernel<E, decltype(u)::value>), grid, dim3(256), 0, stream, x, r, xo, g, p.eps, y,
                           p.values, p.scales, p.dim, Kp);
    };
    if (units <= 256) go(std::integral_constant<int, 1>{});
    else if (units <= 512) go(std::integral_constant<int, 2>{});
    else if (units <= 1024) go(std::integral_constant<int, 4>{});
    else go(std::integral_constant<int, 8>{});
    return hipGetLastError();
}

}  // namespace

hipError_t mx_quantize(int dtype, const MxQuantize &p, hipStream_t stream) {
    if (dtype == 1) return quantize_t<__bf16>(p, stream);
    if (dtype == 2) return quantize_t<_Float16>(p, stream);
    return quantize_t<float>(p, stream);
}

hipError_t mx_rms_norm(int dtype, const MxNorm &p, hipStream_t stream) {
    if (dtype == 1) return norm_t<__bf16>(p, stream);
    if (dtype == 2) return norm_t<_Float16>(p, stream);
    return norm_t<float>(p, stream);
}

}  // namespace vgdr
