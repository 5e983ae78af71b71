// Products of rows with 4-bit weights (gdr_mx.hpp): y[b][n] = sum_k x[b][k] w[n][k], and for a gated pair of weights
// silu(x W1^T) (x W2^T).
//
// Rows in 8 bits meet the weights in v_mfma_scale_f32_16x16x128_f8f6f4, which takes both formats and both
// blocks' scales as they lie.  bf16 rows meet them in v_mfma_f32_16x16x32_bf16 after
// v_cvt_scalef32_pk_bf16_fp4, exactly: a 4-bit value times a power of two is a bf16 number.  The weights
// are the products' A operand, so a lane (g, r) ends up with weight rows 4 g .. + 3 of a
// tile for row r of x: neighbouring columns of y.
//
// A K tile is 128 columns.  Lane (g, r) holds of its 16 weight rows' tile row r, columns 32 g .. + 31 (16 bytes,
// one coalesced KB a wave), and of the rows' tile
//   8 bits:  row r, bytes 16 g .. + 15 and 64 + 16 g .. + 15 (the instruction's order), the scale of block g;
//   bf16:    row r, columns 32 g + 8 i .. + 7 for the products i = 0 .. 3 (any order that both operands share).
#include "gdr_kernels.hpp"
#include "gdr_mx.hpp"

namespace vgdr {

namespace {

// the four bf16 pairs of eight 4-bit values
__device__ __forceinline__ bf16x8 to_bf16(uint32_t q, float scale) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 0);
    const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 1);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 2);
    const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 3);
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// 4-bit rows of A, 8-bit rows of B, their blocks' scale bytes
__device__ __forceinline__ f32x4 mfma_mx(u32x4 w, int ws, u32x4 lo, u32x4 hi, int xs, f32x4 c) {
    const i32x8 a = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
    const i32x8 b = {(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 4, 0, 0, ws, 0, xs);
}

// silu(a) b.  Where the result is rounded to 16 or 8 bits, by the hardware's exponential and
// reciprocal (a few 2^-23); fp32 results take the accurate ones, which cost an epilogue three times as much.
__device__ __forceinline__ float gated_product(float a, float b, bool accurate) {
    if (accurate) return a / (1.f + expf(-a)) * b;
    return a * sigmoidf_(a) * b;
}

// y[row][col .. col + 3] in type `out`; columns from N on are dropped
__device__ __forceinline__ void store4(const MxLinear &p, int64_t row, int col, f32x4 v) {
    if (row >= p.rows || col >= p.N) return;
    const int64_t at = row * p.N + col;
    const bool whole = (p.N & 3) == 0;                                // and col + 3 < N, the address aligned
    if (p.out == 0) {
        float *y = reinterpret_cast<float *>(p.y) + at;
        if (whole) {
            *reinterpret_cast<f32x4 *>(y) = v;
            return;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (col + j < p.N) y[j] = v[j];
    } else if (p.out == 1) {
        __bf16 *y = reinterpret_cast<__bf16 *>(p.y) + at;
        const bf16x4 o = Elem<__bf16>::cvt(v);
        if (whole) {
            *reinterpret_cast<bf16x4 *>(y) = o;
            return;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (col + j < p.N) y[j] = o[j];
    } else {
        _Float16 *y = reinterpret_cast<_Float16 *>(p.y) + at;
        const f16x4 o = Elem<_Float16>::cvt(v);
        if (whole) {
            *reinterpret_cast<f16x4 *>(y) = o;
            return;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (col + j < p.N) y[j] = o[j];
    }
}

// The results of one tile of 16 rows and MT consecutive weight tiles from tile t0 on, acc[MT].
template <bool GATED, int MT>
__device__ __forceinline__ void epilogue(const MxLinear &p, int64_t row, int t0, int g, const f32x4 *acc) {
    if constexpr (!GATED) {
#pragma unroll
        for (int a = 0; a < MT; ++a)
            if (t0 + a < p.T) store4(p, row, 16 * (t0 + a) + 4 * g, acc[a]);
    } else {
        f32x4 v[MT / 2];
#pragma unroll
        for (int a = 0; a < MT / 2; ++a)
#pragma unroll
            for (int j = 0; j < 4; ++j) v[a][j] = gated_product(acc[2 * a][j], acc[2 * a + 1][j], p.out == 0);
        if (p.out != MX8) {
#pragma unroll
            for (int a = 0; a < MT / 2; ++a)
                if (t0 + 2 * a < p.T) store4(p, row, 8 * t0 + 16 * a + 4 * g, v[a]);
            return;
        }
        if constexpr (MT % 4 == 0) {
            // two pairs of tiles are a block of 32 columns, whose values are in the four lanes of row r
            const int64_t Np = (p.N + 127) / 128 * 128;
#pragma unroll
            for (int q = 0; q < MT / 4; ++q) {
                uint32_t amax = 0;
                float f[2][4];
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        f[h][j] = t0 + 4 * q + 2 * h < p.T ? v[2 * q + h][j] : 0.f;   // past the weights: padding
                        amax = max(amax, abs_bits(f[h][j]));
                    }
                amax = max(amax, (uint32_t)__shfl_xor((int)amax, 16));
                amax = max(amax, (uint32_t)__shfl_xor((int)amax, 32));
                const int b = mx_scale<8>(amax), col = 8 * t0 + 32 * q;
                if (row < p.rows && col < Np) {
                    uint8_t *y = reinterpret_cast<uint8_t *>(p.y) + row * Np + col + 4 * g;
#pragma unroll
                    for (int h = 0; h < 2; ++h) *reinterpret_cast<uint32_t *>(y + 16 * h) = mx_pack8(f[h], b);
                    if (g == 0) p.y_scales[(row * Np + col) / 32] = (uint8_t)b;
                }
            }
        }
    }
}

}  // namespace

// Few rows: a workgroup owns MT weight tiles and 16 NB rows; its NWV waves take every NWV-th K tile and
// meet in LDS, in a fixed order.  A wave stages its rows' tiles through an LDS region of its own (a load
// covers whole rows, and no barrier is needed for it).
template <bool X8, bool GATED, int MT, int NB, int NWV>
__global__ void __launch_bounds__(64 * NWV) mx_few_rows_kernel(const MxLinear p) {
    constexpr int ROW = X8 ? 128 : 256, PITCH = ROW + 16, LR = 1024 / ROW, NL = 16 * NB / LR;
    constexpr int STAGE = 16 * NB * PITCH, RED = NWV / 2 * MT * NB * 64 * 16;
    constexpr int LDS = STAGE * NWV > RED ? STAGE * NWV : RED;
    __shared__ __attribute__((aligned(16))) char lds[LDS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, r = lane & 15;
    const int t0 = blockIdx.x * MT;
    const int64_t b0 = (int64_t)blockIdx.y * 16 * NB;
    const int C4 = (p.C + 3) / 4;

    const uint8_t *w[MT], *ws[MT];
#pragma unroll
    for (int a = 0; a < MT; ++a) {
        const int t = t0 + a < p.T ? t0 + a : p.T - 1;
        w[a] = p.w + (int64_t)t * p.C * 1024 + lane * 16;
        ws[a] = p.w_scales + (int64_t)t * C4 * 256 + lane * 4;
    }
    // a lane loads 16 bytes of row lane / (64 / LR) + LR i; rows past the end are the last one again
    const int lr = lane / (64 / LR), lk = lane % (64 / LR) * 16;
    const char *src[NL];
#pragma unroll
    for (int i = 0; i < NL; ++i) {
        const int64_t row = b0 + LR * i + lr < p.rows ? b0 + LR * i + lr : p.rows - 1;
        src[i] = reinterpret_cast<const char *>(p.x) + row * p.ldx * (X8 ? 1 : 2) + lk;
    }
    const uint8_t *xs[NB];
    if constexpr (X8) {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int64_t row = b0 + 16 * b + r < p.rows ? b0 + 16 * b + r : p.rows - 1;
            xs[b] = p.x_scales + row * 4 * p.C + g;
        }
    }
    const int64_t plane = X8 ? 0 : p.rows * p.ldx * 2;

    f32x4 acc[MT][NB];
#pragma unroll
    for (int a = 0; a < MT; ++a)
#pragma unroll
        for (int b = 0; b < NB; ++b) acc[a][b] = f32x4{0.f, 0.f, 0.f, 0.f};

    // step s: K tile wave + NWV (s / planes), plane s % planes
    const int mine = wave < p.C ? (p.C - wave + NWV - 1) / NWV : 0;
    u32x4 wn[MT], xn[NL];
    int wsn[MT], xsn[NB];
    auto load = [&](int c, int plane_at) __attribute__((always_inline)) {
#pragma unroll
        for (int a = 0; a < MT; ++a) {
            wn[a] = *reinterpret_cast<const u32x4 *>(w[a] + (int64_t)c * 1024);
            wsn[a] = ws[a][(c >> 2) * 256 + (c & 3)];
        }
#pragma unroll
        for (int i = 0; i < NL; ++i) xn[i] = *reinterpret_cast<const u32x4 *>(src[i] + plane_at * plane + (int64_t)c * ROW);
        if constexpr (X8) {
#pragma unroll
            for (int b = 0; b < NB; ++b) xsn[b] = xs[b][4 * c];
        }
    };
    char *stage = lds + wave * STAGE;
    const int steps = mine * p.planes;
    int c = wave, pl = 0;
    if (steps) load(c, 0);
    for (int s = 0; s < steps; ++s) {
        u32x4 wc[MT];
        int wsc[MT], xsc[NB];
#pragma unroll
        for (int a = 0; a < MT; ++a) {
            wc[a] = wn[a];
            wsc[a] = wsn[a];
        }
        if constexpr (X8) {
#pragma unroll
            for (int b = 0; b < NB; ++b) xsc[b] = xsn[b];
        }
#pragma unroll
        for (int i = 0; i < NL; ++i) *reinterpret_cast<u32x4 *>(stage + (LR * i + lr) * PITCH + lk) = xn[i];
        // the region is this wave's alone: LDS operations of one wave are in order, and only the compiler has to keep it
        asm volatile("" ::: "memory");
        if (++pl == p.planes) {
            pl = 0;
            c += NWV;
        }
        if (s + 1 < steps) load(c, pl);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const char *at = stage + (16 * b + r) * PITCH;
            if constexpr (X8) {
                const u32x4 lo = *reinterpret_cast<const u32x4 *>(at + 16 * g);
                const u32x4 hi = *reinterpret_cast<const u32x4 *>(at + 64 + 16 * g);
#pragma unroll
                for (int a = 0; a < MT; ++a) acc[a][b] = mfma_mx(wc[a], wsc[a], lo, hi, xsc[b], acc[a][b]);
            } else {
                bf16x8 f[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) f[i] = *reinterpret_cast<const bf16x8 *>(at + 64 * g + 16 * i);
#pragma unroll
                for (int a = 0; a < MT; ++a) {
                    const float scale = mx_value(wsc[a]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[a][b] = mfma_pair(to_bf16(wc[a][i], scale), f[i], acc[a][b]);
                }
            }
        }
        asm volatile("" ::: "memory");
    }
    // the waves' sums, halves onto halves
    f32x4 *red = reinterpret_cast<f32x4 *>(lds);
#pragma unroll
    for (int half = NWV / 2; half > 0; half /= 2) {
        __syncthreads();
        if (wave >= half && wave < 2 * half) {
#pragma unroll
            for (int a = 0; a < MT; ++a)
#pragma unroll
                for (int b = 0; b < NB; ++b) red[(((wave - half) * MT + a) * NB + b) * 64 + lane] = acc[a][b];
        }
        __syncthreads();
        if (wave < half) {
#pragma unroll
            for (int a = 0; a < MT; ++a)
#pragma unroll
                for (int b = 0; b < NB; ++b) acc[a][b] += red[((wave * MT + a) * NB + b) * 64 + lane];
        }
    }
    if (wave > 0) return;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        f32x4 v[MT];
#pragma unroll
        for (int a = 0; a < MT; ++a) v[a] = acc[a][b];
        epilogue<GATED, MT>(p, b0 + 16 * b + r, t0, g, v);
    }
}

// Many rows: a workgroup owns BM rows and BN / 16 weight tiles, its WM x WN waves BM / WM x BN / WN each.  The rows'
// K tiles go to LDS asynchronously, NBUF - 1 steps ahead, in 16-byte units swizzled so that the 16
// rows of a fragment lie on distinct banks; a wave loads its weights' fragments from global memory, a step
// ahead: they lie there as it needs them.
template <bool X8, bool GATED, int BM, int BN, int WM, int WN, int NBUF>
__global__ void __launch_bounds__(64 * WM * WN) mx_tile_kernel(const MxLinear p, int mb, int nb) {
    constexpr int ROW = X8 ? 128 : 256, UPR = ROW / 16, NWV = WM * WN;
    constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
    constexpr int DMAS = BM * ROW / 1024 / NWV;                       // a wave's copies of a step
    static_assert(BM * ROW % (1024 * NWV) == 0 && BM % 64 == 0, "whole copies");
    static_assert(!X8 || BM / 64 <= NWV, "a wave copies the scales of 64 rows");
    __shared__ __attribute__((aligned(16))) char xb[NBUF][BM * ROW];
    __shared__ __attribute__((aligned(16))) uint32_t xsb[X8 ? NBUF : 1][X8 ? BM : 4];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, r = lane & 15, wm = wave / WN, wn = wave % WN;

    // an XCD (every eighth workgroup) walks a run of its own of the tiles, eight row blocks under each column block:
    // its L2 holds those rows and meets every weight once for eight blocks
    const int64_t total = (int64_t)mb * nb, per = (total + 7) / 8;
    const int64_t id = (int64_t)(blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if ((blockIdx.x >> 3) >= per || id >= total) return;
    const int64_t band = id / (8 * (int64_t)nb);
    const int high = mb - band * 8 < 8 ? (int)(mb - band * 8) : 8;
    const int64_t in = id - band * 8 * nb;
    const int64_t m0 = (band * 8 + in % high) * BM;
    const int t0 = (int)(in / high) * (BN / 16) + wn * FN;

    const int C4 = (p.C + 3) / 4;
    const uint8_t *w[FN], *ws[FN];
#pragma unroll
    for (int a = 0; a < FN; ++a) {
        const int t = t0 + a < p.T ? t0 + a : p.T - 1;
        w[a] = p.w + (int64_t)t * p.C * 1024 + lane * 16;
        ws[a] = p.w_scales + (int64_t)t * C4 * 256 + lane * 4;
    }
    // copy i of this wave fills units 64 (wave DMAS + i) .. + 63 of the tile; unit u of row R lies at u ^ swz(R)
    auto swz = [](int R) { return X8 ? (R >> 1) & 7 : R & 15; };
    const char *src[DMAS];
#pragma unroll
    for (int i = 0; i < DMAS; ++i) {
        const int at = 64 * (wave * DMAS + i) + lane, R = at / UPR, u = at % UPR ^ swz(R);
        const int64_t row = m0 + R < p.rows ? m0 + R : p.rows - 1;
        src[i] = reinterpret_cast<const char *>(p.x) + row * p.ldx * (X8 ? 1 : 2) + u * 16;
    }
    // every wave copies the scales of 64 rows, so that all have as many copies on their way: where there are
    // more waves than that, some copy the same
    const int sblock = wave % (BM / 64);
    const uint8_t *xsrc = nullptr;
    if constexpr (X8) {
        const int64_t row = m0 + 64 * sblock + lane < p.rows ? m0 + 64 * sblock + lane : p.rows - 1;
        xsrc = p.x_scales + row * 4 * p.C;
    }
    const int64_t plane = X8 ? 0 : p.rows * p.ldx * 2;
    const int steps = p.C * p.planes;

    int ic = 0, ip = 0, is = 0;                                       // the next copy's K tile, plane and buffer
    auto copy = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < DMAS; ++i)
            lds_dma16(src[i] + ip * plane + (int64_t)ic * ROW, xb[is] + (wave * DMAS + i) * 1024);
        if constexpr (X8) lds_dma4(xsrc + 4 * (int64_t)ic, xsb[is] + 64 * sblock);
        if (++ip == p.planes) {
            ip = 0;
            ++ic;
        }
        is = is + 1 == NBUF ? 0 : is + 1;
    };

    f32x4 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int a = 0; a < FN; ++a) acc[i][a] = f32x4{0.f, 0.f, 0.f, 0.f};
    u32x4 wn_[FN];
    int wsn[FN];
    auto load = [&](int c) __attribute__((always_inline)) {
#pragma unroll
        for (int a = 0; a < FN; ++a) {
            wn_[a] = *reinterpret_cast<const u32x4 *>(w[a] + (int64_t)c * 1024);
            wsn[a] = ws[a][(c >> 2) * 256 + (c & 3)];
        }
    };
    load(0);
#pragma unroll
    for (int s = 0; s < NBUF - 1; ++s)
        if (s < steps) copy();
    int c = 0, pl = 0, buf = 0;
    for (int s = 0; s < steps; ++s) {
        // this step's copies have landed: of this wave's copies only those of the NBUF - 2 steps after it may
        // still be on their way (loads that the compiler places in between make the wait longer, never shorter)
        if (NBUF > 2 && s + NBUF - 2 < steps)
            asm volatile("s_waitcnt vmcnt(%0)" :: "n"((NBUF - 2) * (DMAS + (X8 ? 1 : 0))) : "memory");
        else
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        lds_barrier();
        u32x4 wc[FN];
        int wsc[FN];
#pragma unroll
        for (int a = 0; a < FN; ++a) {
            wc[a] = wn_[a];
            wsc[a] = wsn[a];
        }
        if (++pl == p.planes) {
            pl = 0;
            ++c;
        }
        if (s + 1 < steps) load(c);
        if (s + NBUF - 1 < steps) copy();
        const char *tile = xb[buf];
        if constexpr (X8) {
#pragma unroll
            for (int i = 0; i < FM; ++i) {
                const int R = (wm * FM + i) * 16 + r;
                const u32x4 lo = *reinterpret_cast<const u32x4 *>(tile + R * ROW + (g ^ swz(R)) * 16);
                const u32x4 hi = *reinterpret_cast<const u32x4 *>(tile + R * ROW + ((4 + g) ^ swz(R)) * 16);
                const int xs = reinterpret_cast<const uint8_t *>(xsb[buf] + R)[g];
#pragma unroll
                for (int a = 0; a < FN; ++a) acc[i][a] = mfma_mx(wc[a], wsc[a], lo, hi, xs, acc[i][a]);
            }
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                bf16x8 f[FN];
#pragma unroll
                for (int a = 0; a < FN; ++a) f[a] = to_bf16(wc[a][k], mx_value(wsc[a]));
#pragma unroll
                for (int i = 0; i < FM; ++i) {
                    const int R = (wm * FM + i) * 16 + r;
                    const bf16x8 x = *reinterpret_cast<const bf16x8 *>(tile + R * ROW + ((4 * g + k) ^ swz(R)) * 16);
#pragma unroll
                    for (int a = 0; a < FN; ++a) acc[i][a] = mfma_pair(f[a], x, acc[i][a]);
                }
            }
        }
        buf = buf + 1 == NBUF ? 0 : buf + 1;
    }
#pragma unroll
    for (int i = 0; i < FM; ++i) epilogue<GATED, FN>(p, m0 + (wm * FM + i) * 16 + r, t0, g, acc[i]);
}

namespace {

template <bool X8, bool GATED, int MT, int NB, int NWV>
hipError_t few_rows_go(const MxLinear &p, int tiles, hipStream_t stream) {
    const dim3 grid((unsigned)((tiles + MT - 1) / MT), (unsigned)((p.rows + 16 * NB - 1) / (16 * NB)));
    hipLaunchKernelGGL((mx_few_rows_kernel<X8, GATED, MT, NB, NWV>), grid, dim3(64 * NWV), 0, stream, p);
    return hipGetLastError();
}

template <bool X8, bool GATED, int BM, int BN, int WM, int WN, int NBUF>
hipError_t tile_go(const MxLinear &p, int tiles, hipStream_t stream) {
    const int64_t mb = (p.rows + BM - 1) / BM, nb = (tiles + BN / 16 - 1) / (BN / 16);
    const int64_t blocks = (mb * nb + 7) / 8 * 8;
    hipLaunchKernelGGL((mx_tile_kernel<X8, GATED, BM, BN, WM, WN, NBUF>), dim3((unsigned)blocks), dim3(64 * WM * WN), 0, stream,
                       p, (int)mb, (int)nb);
    return hipGetLastError();
}

template <bool X8, bool GATED>
hipError_t mx_linear_t(const MxLinear &p, hipStream_t stream) {
    // the output's padding to whole 128s of columns counts as tiles (8-bit outputs: 8 pairs a 128)
    const int tiles = GATED && p.out == MX8 ? (p.N + 127) / 128 * 16 : p.T;
    if (p.rows <= 16) return few_rows_go<X8, GATED, GATED ? 4 : 1, 1, 8>(p, tiles, stream);
    if (p.rows <= 64) return few_rows_go<X8, GATED, GATED ? 4 : 1, 4, 8>(p, tiles, stream);
    const int64_t cus = device_cu_count();
    if ((p.rows + 255) / 256 * ((tiles + 15) / 16) >= cus) {
        if constexpr (X8) return tile_go<X8, GATED, 256, 256, 2, 4, 3>(p, tiles, stream);
        else return tile_go<X8, GATED, 256, 256, 2, 4, 2>(p, tiles, stream);
    }
    return tile_go<X8, GATED, 64, 128, 2, 2, 3>(p, tiles, stream);
}

}  // namespace

hipError_t mx_linear(const MxLinear &p, hipStream_t stream) {
    if (p.x8) return p.gated ? mx_linear_t<true, true>(p, stream) : mx_linear_t<true, false>(p, stream);
    return p.gated ? mx_linear_t<false, true>(p, stream) : mx_linear_t<false, false>(p, stream);
}

}  // namespace vgdr
