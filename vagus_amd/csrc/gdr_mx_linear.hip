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

// 4-bit rows of A, 8-bit rows of B, their blocks' scale bytes.  The instruction sums its 128 products in fewer bits than fp32
// (results off by 1.2e-5 rms at K 128 to 8192; bf16 rows 1e-8 to 1.3e-7) and adds to fp32.  Taken for its rate, twice bf16's: the
// rows' rounding to 8 bits is off by 2.6e-2 of a result, 2,000 times that.
__device__ __forceinline__ f32x4 mfma_mx(u32x4 w, int ws, u32x4 lo, u32x4 hi, int xs, f32x4 c) {
    const i32x8 a = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
    const i32x8 b = {(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 4, 0, 0, ws, 0, xs);
}

// Behind the loop of matrix instructions: whichever way the loop was left, their results pass their wait states here
// before anything reads them.  Tied to the accumulators instead, it cost the largest products 4 %.
__device__ __forceinline__ void settle() {
    asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// silu(a) b.  Where the result is rounded to 16 bits, or the sums are those of 8-bit rows, by the hardware's exponential and
// reciprocal (a few 2^-23).  fp32 results take the accurate ones, which cost an epilogue three times as much, and so do 8-bit
// results of 16- and 32-bit rows, whose blocks' scales hang on the last bits of an fp32 sum (4096 rows, gated 11264, K 2048 of
// bf16 to 8 bits: 168 us, 158 without).
__device__ __forceinline__ float gated_product(float a, float b, bool accurate) {
    if (accurate) return a / (1.f + expf(-a)) * b;
    return a * sigmoidf_(a) * b;
}

// y[row][col .. col + 4 V - 1] in type `out`; columns from N on are dropped
template <typename E, int V>
__device__ __forceinline__ void store_as(const MxLinear &p, int64_t row, int col, const f32x4 *v) {
    typedef E EV __attribute__((ext_vector_type(4 * V)));
    E *y = reinterpret_cast<E *>(p.y) + row * p.N + col;
    EV o;
#pragma unroll
    for (int j = 0; j < 4 * V; ++j) o[j] = (E)v[j / 4][j % 4];
    if (col + 4 * V <= p.N) {                                         // whole, at whatever address N makes it
        __builtin_memcpy(y, &o, sizeof o);
        return;
    }
#pragma unroll
    for (int j = 0; j < 4 * V; ++j)
        if (col + j < p.N) y[j] = o[j];
}
template <int V>
__device__ __forceinline__ void store(const MxLinear &p, int64_t row, int col, const f32x4 *v) {
    if (row >= p.rows || col >= p.N) return;
    if (p.out == 0) store_as<float, V>(p, row, col, v);
    else if (p.out == 1) store_as<__bf16, V>(p, row, col, v);
    else store_as<_Float16, V>(p, row, col, v);
}

// Which weight row MFMA row r of weight tile a meets, of the MT tiles from t0 on.  Results come out four
// to a lane, of the rows 4 g .. + 3 of a tile; two tiles of the same kind (of the same weight, where they are gated) are
// taken as 32 rows of which MFMA row 4 g + j of the h-th is row 8 g + 4 h + j, so that a lane ends up with eight
// neighbouring columns, a row of y with 64 bytes in one store, and an 8-bit block with eight bytes a lane.
struct WeightRow {
    int tile, row;
};
template <bool GATED, int MT>
__device__ __forceinline__ WeightRow weight_row(int a, int t0, int r) {
    if constexpr (MT == 1) return {t0, r};
    const int h = GATED ? a / 2 % 2 : a % 2;
    const int first = GATED ? t0 + a / 4 * 4 + a % 2 : t0 + a / 2 * 2;
    return {first + (r >> 3) * (GATED ? 2 : 1), 8 * (r >> 2 & 1) + 4 * h + (r & 3)};
}

// The results of row `row` (MFMA column r) from the MT weight tiles from t0 on, acc[MT].
template <bool GATED, int MT>
__device__ __forceinline__ void epilogue(const MxLinear &p, int64_t row, int t0, int g, const f32x4 *acc) {
    if constexpr (!GATED) {
        if constexpr (MT == 1) {
            store<1>(p, row, 16 * t0 + 4 * g, acc);
        } else {
#pragma unroll
            for (int q = 0; q < MT / 2; ++q) store<2>(p, row, 16 * (t0 + 2 * q) + 8 * g, acc + 2 * q);
        }
    } else {
        static_assert(MT % 4 == 0, "two pairs of gated tiles are a block of 32 columns");
#pragma unroll
        for (int q = 0; q < MT / 4; ++q) {
            f32x4 v[2];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    v[h][j] = gated_product(acc[4 * q + 2 * h][j], acc[4 * q + 2 * h + 1][j], p.accurate);
            const int col = 8 * (t0 + 4 * q) + 8 * g;
            if (p.out != MX8) {
                store<2>(p, row, col, v);
                continue;
            }
            const int64_t Np = (p.N + 127) / 128 * 128;
            uint32_t amax = 0;
            float f[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                f[j] = col + j < p.N ? v[j / 4][j % 4] : 0.f;                       // past the weights: padding
                amax = max(amax, abs_bits(f[j]));
            }
            amax = max(amax, (uint32_t)__shfl_xor((int)amax, 16));
            amax = max(amax, (uint32_t)__shfl_xor((int)amax, 32));
            const int b = mx_scale<8>(amax);
            if (row < p.rows && col < Np) {
                *reinterpret_cast<u32x2 *>(reinterpret_cast<uint8_t *>(p.y) + row * Np + col) = u32x2{mx_pack8(f, b), mx_pack8(f + 4, b)};
                if (g == 0) p.y_scales[(row * Np + col) / 32] = (uint8_t)b;
            }
        }
    }
}

}  // namespace

constexpr int BF16_TAIL = 4;

// Few rows: a workgroup owns MT weight tiles and 16 NB rows; its NWV waves take every NWV-th K tile, the next one's loads
// ahead of this one's products, and meet in LDS, in a fixed order.  A wave passes its rows' tiles through an LDS
// region of its own, which needs no barrier: a load covers whole rows of a tile there, where fragments
// straight from global memory would have every lane in a line of its own, and the address unit bounds those
// (64 rows, K 5632, N 2048: 9.6 us, 5.9 through LDS; 64 rows, K and N 8192: 25, 17.7).
// Bound by latency, a chain of launch, first loads, K / 128 / NWV steps and the meeting in LDS.  Recorded, with the weights in the
// caches / from memory, as a model's step finds them: one row, K 2048, N 8192 3.7 / 5.0 us (8.9 MB of weights, 1.8 us at a copy's
// rate), 64 rows 7.4 / 8.5; one row, gated 11264, 5.1 / 6.4, 64 rows 9.7 / 11.5.  A longer way ahead in the loads, sixteen
// waves, or eight weight tiles a workgroup took as long or longer.
// X: the rows' type (0 fp32, 1 bf16, 2 fp16, MX8, BF16_TAIL).  fp32 and fp16 rows become three and two bf16 planes on their way
// into LDS; their K, and BF16_TAIL's, may end inside a tile (a check that costs the others half a microsecond).
template <int X, bool GATED, int MT, int NB, int NWV>
__global__ void __launch_bounds__(64 * NWV, 2) mx_few_rows_kernel(const MxLinear p) {
    typedef std::conditional_t<X == 0, float, std::conditional_t<X == 1 || X == BF16_TAIL, __bf16, std::conditional_t<X == 2, _Float16, uint8_t>>> E;
    constexpr bool X8 = X == MX8;
    constexpr int ES = (int)sizeof(E), VE = 16 / ES, P = X == 0 ? 3 : X == 2 ? 2 : 1;
    constexpr int ROW = 128 * ES, LR = 1024 / ROW, NX = 16 * NB / LR;
    constexpr int PITCH = (X8 ? 128 : 256) + 16, PLANE = 16 * NB * PITCH;
    constexpr int STAGE = P * PLANE, RED = NWV / 2 * MT * NB * 64 * 16;
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
        const WeightRow at = weight_row<GATED, MT>(a, t0, r);
        const int64_t t = at.tile < p.T ? at.tile : p.T - 1;            // past the end: the last one again, not stored
        w[a] = p.w + t * p.C * 1024 + (16 * g + at.row) * 16;
        ws[a] = p.w_scales + t * C4 * 256 + (16 * g + at.row) * 4;
    }
    // a lane loads 16 bytes of row lane / (64 / LR) + LR i; rows past the end are the last one again
    const int lr = lane / (64 / LR), lk = lane % (64 / LR) * VE;
    const E *x[NX];
#pragma unroll
    for (int i = 0; i < NX; ++i) {
        const int64_t row = b0 + LR * i + lr < p.rows ? b0 + LR * i + lr : p.rows - 1;
        x[i] = reinterpret_cast<const E *>(p.x) + row * p.ldx + lk;
    }
    const uint8_t *xs[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const int64_t row = b0 + 16 * b + r < p.rows ? b0 + 16 * b + r : p.rows - 1;
        xs[b] = X8 ? p.x_scales + row * 4 * p.C + g : nullptr;
    }
    const int64_t plane = p.rows * p.ldx;                             // of bf16 rows that are planes already
    // Of fp32 and fp16, loads whose rows are all past the end are left out with their conversions (one row of fp32, K 7680,
    // N 2048: 10.4 us, 26.9 with them): those columns of the products are never stored.  bf16 and 8-bit
    // rows repeat the last row instead: the branches cost more (16 rows, K 2048, N 8192: 7.1 us against 6.5).
    const int live = P > 1 && p.rows - b0 < 16 * NB ? (int)(p.rows - b0) : 16 * NB;

    f32x4 acc[MT][NB];
#pragma unroll
    for (int a = 0; a < MT; ++a)
#pragma unroll
        for (int b = 0; b < NB; ++b) acc[a][b] = f32x4{0.f, 0.f, 0.f, 0.f};

    struct Step {
        u32x4 w[MT], x[NX];
        int ws[MT], xs[NB];
    };
    // step s: K tile wave + NWV (s / planes), plane s % planes
    const int steps = (wave < p.C ? (p.C - wave + NWV - 1) / NWV : 0) * p.planes;
    int c = wave, pl = 0;
    auto load = [&](Step &to) __attribute__((always_inline)) {
#pragma unroll
        for (int a = 0; a < MT; ++a) {
            to.w[a] = *reinterpret_cast<const u32x4 *>(w[a] + (int64_t)c * 1024);
            to.ws[a] = ws[a][(c >> 2) * 256 + (c & 3)];
        }
        if (X8 || X == 1 || 128 * (c + 1) <= p.K) {
#pragma unroll
            for (int i = 0; i < NX; ++i)
                if (P == 1 || LR * i < live) to.x[i] = *reinterpret_cast<const u32x4 *>(x[i] + pl * plane + 128 * (int64_t)c);
        } else {
            typedef E V __attribute__((ext_vector_type(VE)));
#pragma unroll
            for (int i = 0; i < NX; ++i) {
                if (P > 1 && LR * i >= live) break;
                V v;
#pragma unroll
                for (int e = 0; e < VE; ++e) v[e] = 128 * c + lk + e < p.K ? x[i][pl * plane + 128 * (int64_t)c + e] : (E)0;
                to.x[i] = __builtin_bit_cast(u32x4, v);
            }
        }
        if constexpr (X8) {
#pragma unroll
            for (int b = 0; b < NB; ++b) to.xs[b] = xs[b][4 * (int64_t)c];
        }
        if (++pl == p.planes) {
            pl = 0;
            c += NWV;
        }
    };
    char *stage = lds + wave * STAGE;
    auto put = [&](const Step &of) __attribute__((always_inline)) {
        // LDS operations of one wave are in order: only the compiler has to keep it
        asm volatile("" ::: "memory");
#pragma unroll
        for (int i = 0; i < NX; ++i) {
            if (P > 1 && LR * i >= live) break;
            char *to = stage + (LR * i + lr) * PITCH + lk * (X8 ? 1 : 2);
            if constexpr (P == 1) {
                *reinterpret_cast<u32x4 *>(to) = of.x[i];
            } else {
                typedef E V __attribute__((ext_vector_type(VE)));
                typedef __bf16 O __attribute__((ext_vector_type(VE)));
                const V v = __builtin_bit_cast(V, of.x[i]);
                O o[P];
#pragma unroll
                for (int e = 0; e < VE; ++e) {
                    __bf16 part[P];
                    split(part, (float)v[e]);
#pragma unroll
                    for (int q = 0; q < P; ++q) o[q][e] = part[q];
                }
#pragma unroll
                for (int q = 0; q < P; ++q) *reinterpret_cast<O *>(to + q * PLANE) = o[q];
            }
        }
        asm volatile("" ::: "memory");
    };
    auto products = [&](const Step &of) __attribute__((always_inline)) {
        if constexpr (X8) {
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const char *at = stage + (16 * b + r) * PITCH + 16 * g;
                const u32x4 lo = *reinterpret_cast<const u32x4 *>(at), hi = *reinterpret_cast<const u32x4 *>(at + 64);
#pragma unroll
                for (int a = 0; a < MT; ++a) acc[a][b] = mfma_mx(of.w[a], of.ws[a], lo, hi, of.xs[b], acc[a][b]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                bf16x8 f[P][NB];
#pragma unroll
                for (int q = 0; q < P; ++q)
#pragma unroll
                    for (int b = 0; b < NB; ++b)
                        f[q][b] = *reinterpret_cast<const bf16x8 *>(stage + q * PLANE + (16 * b + r) * PITCH + 64 * g + 16 * i);
#pragma unroll
                for (int a = 0; a < MT; ++a) {
                    const bf16x8 v = to_bf16(of.w[a][i], mx_value(of.ws[a]));
#pragma unroll
                    for (int q = 0; q < P; ++q)
#pragma unroll
                        for (int b = 0; b < NB; ++b) acc[a][b] = mfma_pair(v, f[q][b], acc[a][b]);
                }
            }
        }
    };
    Step even, odd;
    if (steps > 0) load(even);
    for (int s = 0; s < steps; s += 2) {
        put(even);
        if (s + 1 < steps) load(odd);
        products(even);
        if (s + 1 == steps) break;
        put(odd);
        if (s + 2 < steps) load(even);
        products(odd);
    }
    settle();
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

// Many rows: a workgroup owns BM rows and BN / 16 weight tiles, its WM x WN waves BM / WM x BN / WN each.  The K tiles of
// both go to LDS asynchronously, a step ahead.  In LDS a row of x is cut into 16-byte units whose places
// are swizzled so that the 16 rows of a fragment lie on distinct banks; of the two weight tiles that
// weight_row mixes the second has its rows' places moved by four for the same reason.
// Two workgroups share a CU: one's barriers, first copies and stores lie under the other's products.  At K = 2048
// that is the larger part: 65,536 rows in 8 bits, N 8192: 925 us (2,380 TFLOP/s); one workgroup of 256 x 256 and
// three stages 1,240, its next tile's copies begun under the stores 1,220; at K = N = 8192, 16,384 rows 790 us
// (2,780 TFLOP/s) against 880.  The weights' fragments straight from global memory into registers: 1,360
// (the wait for them is a wait for the copies behind them too).  bf16 rows: 1,730 us (1,270 TFLOP/s); there the LDS
// for two workgroups allows 64 x 256, and the conversions share the issue slots with twice the products' time.
template <bool X8, bool GATED, int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(64 * WM * WN, 2 * WM * WN / 4) mx_tile_kernel(const MxLinear p, uint32_t mb, uint32_t nb) {
    constexpr int ROW = X8 ? 128 : 256, UPR = ROW / 16, NWV = WM * WN;
    constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
    constexpr uint32_t BAND = 8;
    constexpr int DX = BM * ROW / 1024 / NWV, DW = BN / 16 / NWV;                     // a wave's copies of a step
    static_assert(BM * ROW % (1024 * NWV) == 0 && BN % (16 * NWV) == 0 && BM % 64 == 0 && BN % 64 == 0, "whole copies");
    static_assert(BM / 64 <= NWV && BN / 64 <= NWV, "a wave copies the scales of 64 rows of each");
    struct Stage {
        char x[BM * ROW];
        char w[BN / 16][1024];
        char ws[BN / 16][256];                                        // of four K tiles
        uint32_t xs[X8 ? BM : 4];
    };
    __shared__ __attribute__((aligned(16))) Stage stage[2];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, r = lane & 15, wm = wave / WN, wn = wave % WN;

    // an XCD (every eighth workgroup) walks a run of its own of the tiles, BAND row blocks under each column block: its
    // L2 holds those rows and meets every weight once for BAND blocks
    const uint32_t total = mb * nb, per = (total + 7) / 8, id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if ((blockIdx.x >> 3) >= per || id >= total) return;
    const uint32_t band = id / (BAND * nb), high = mb - band * BAND < BAND ? mb - band * BAND : BAND, in = id - band * BAND * nb;
    const int64_t m0 = (int64_t)(band * BAND + in % high) * BM;
    const int t0 = (int)(in / high) * (BN / 16);

    const int C4 = (p.C + 3) / 4;
    // rows and weights past the end are the last ones again: their results are not stored
    auto swz = [](int R) { return X8 ? (R >> 1) & 7 : R & 15; };      // unit u of row R lies at u ^ swz(R)
    auto moved = [](int t) { return GATED ? (t >> 1 & 1) * 4 : (t & 1) * 4; };
    const char *src[DX + DW], *wsrc, *xsrc = nullptr;
#pragma unroll
    for (int i = 0; i < DX; ++i) {
        const int at = 64 * (wave * DX + i) + lane, R = at / UPR, u = at % UPR ^ swz(R);
        const int64_t row = m0 + R < p.rows ? m0 + R : p.rows - 1;
        src[i] = reinterpret_cast<const char *>(p.x) + row * p.ldx * (X8 ? 1 : 2) + u * 16;
    }
#pragma unroll
    for (int i = 0; i < DW; ++i) {
        const int a = wave * DW + i;
        const int64_t t = t0 + a < p.T ? t0 + a : p.T - 1;
        src[DX + i] = reinterpret_cast<const char *>(p.w) + t * p.C * 1024 + (lane ^ moved(a)) * 16;
    }
    // the scales: where there are more waves than blocks of 64 rows, some copy the same
    const int wblock = wave % (BN / 64), xblock = wave % (BM / 64);
    {
        const int64_t t = t0 + 4 * wblock + g < p.T ? t0 + 4 * wblock + g : p.T - 1;
        wsrc = reinterpret_cast<const char *>(p.w_scales) + t * C4 * 256 + r * 16;
        if constexpr (X8) {
            const int64_t row = m0 + 64 * xblock + lane < p.rows ? m0 + 64 * xblock + lane : p.rows - 1;
            xsrc = reinterpret_cast<const char *>(p.x_scales) + row * 4 * p.C;
        }
    }
    const int64_t plane = X8 ? 0 : p.rows * p.ldx * 2;
    const int steps = p.C * p.planes;

    int ic = 0, ip = 0, is = 0;                                       // the next copy's K tile, plane and stage
    auto copy = [&]() __attribute__((always_inline)) {
        Stage &to = stage[is];
#pragma unroll
        for (int i = 0; i < DX; ++i) lds_dma16(src[i] + ip * plane + (int64_t)ic * ROW, to.x + (wave * DX + i) * 1024);
#pragma unroll
        for (int i = 0; i < DW; ++i) lds_dma16(src[DX + i] + (int64_t)ic * 1024, to.w[wave * DW + i]);
        lds_dma16(wsrc + (int64_t)(ic >> 2) * 256, to.ws[4 * wblock]);
        if constexpr (X8) lds_dma4(xsrc + 4 * (int64_t)ic, to.xs + 64 * xblock);
        if (++ip == p.planes) {
            ip = 0;
            ++ic;
        }
        is ^= 1;
    };

    f32x4 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int a = 0; a < FN; ++a) acc[i][a] = f32x4{0.f, 0.f, 0.f, 0.f};
    // where a lane's weights lie in a stage
    int wat[FN], wsat[FN];
#pragma unroll
    for (int a = 0; a < FN; ++a) {
        const WeightRow at = weight_row<GATED, FN>(a, wn * FN, r);
        wat[a] = at.tile * 1024 + ((16 * g + at.row) ^ moved(at.tile)) * 16;
        wsat[a] = at.tile * 256 + (16 * g + at.row) * 4;
    }
    copy();
    int c = 0, pl = 0;
    for (int s = 0; s < steps; ++s) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");              // this wave's copies of this step have landed
        lds_barrier();                                                // all waves' have, and the last step's stage is read
        if (s + 1 < steps) copy();
        const Stage &from = stage[s & 1];
        u32x4 w[FN];
        int ws[FN];
#pragma unroll
        for (int a = 0; a < FN; ++a) {
            w[a] = *reinterpret_cast<const u32x4 *>(from.w[0] + wat[a]);
            ws[a] = reinterpret_cast<const uint8_t *>(from.ws[0])[wsat[a] + (c & 3)];
        }
        // x's fragments are read one ahead of the products that take them, and stay there: left to the compiler they are
        // read when they are needed (952 us against 917 at 65,536 rows, K 2048, N 8192)
        if constexpr (X8) {
            u32x4 lo[2], hi[2];
            int xs[2];
            auto read = [&](int i) __attribute__((always_inline)) {
                const int R = (wm * FM + i) * 16 + r;
                lo[i & 1] = *reinterpret_cast<const u32x4 *>(from.x + R * ROW + (g ^ swz(R)) * 16);
                hi[i & 1] = *reinterpret_cast<const u32x4 *>(from.x + R * ROW + ((4 + g) ^ swz(R)) * 16);
                xs[i & 1] = reinterpret_cast<const uint8_t *>(from.xs + R)[g];
            };
            read(0);
            unroll<FM>([&](auto ii) __attribute__((always_inline)) {
                constexpr int i = decltype(ii)::value;
                if constexpr (i + 1 < FM) read(i + 1);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int a = 0; a < FN; ++a) acc[i][a] = mfma_mx(w[a], ws[a], lo[i & 1], hi[i & 1], xs[i & 1], acc[i][a]);
            });
        } else {
            bf16x8 x[2];
            auto read = [&](int i) __attribute__((always_inline)) {                  // product i / FM of row tile i % FM
                const int R = (wm * FM + i % FM) * 16 + r;
                x[i & 1] = *reinterpret_cast<const bf16x8 *>(from.x + R * ROW + ((4 * g + i / FM) ^ swz(R)) * 16);
            };
            read(0);
            bf16x8 f[FN];
            unroll<4 * FM>([&](auto ii) __attribute__((always_inline)) {
                constexpr int i = decltype(ii)::value;
                if constexpr (i + 1 < 4 * FM) read(i + 1);
                if constexpr (i % FM == 0) {
#pragma unroll
                    for (int a = 0; a < FN; ++a) f[a] = to_bf16(w[a][i / FM], mx_value(ws[a]));
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int a = 0; a < FN; ++a) acc[i % FM][a] = mfma_pair(f[a], x[i & 1], acc[i % FM][a]);
            });
        }
        if (++pl == p.planes) {
            pl = 0;
            ++c;
        }
    }
    settle();
#pragma unroll
    for (int i = 0; i < FM; ++i) epilogue<GATED, FN>(p, m0 + (wm * FM + i) * 16 + r, t0 + wn * FN, g, acc[i]);
}

namespace {

template <int X, bool GATED, int MT, int NB, int NWV>
hipError_t few_rows_go(const MxLinear &p, int tiles, hipStream_t stream) {
    const dim3 grid((unsigned)((tiles + MT - 1) / MT), (unsigned)((p.rows + 16 * NB - 1) / (16 * NB)));
    hipLaunchKernelGGL((mx_few_rows_kernel<X, GATED, MT, NB, NWV>), grid, dim3(64 * NWV), 0, stream, p);
    return hipGetLastError();
}

template <bool X8, bool GATED, int BM, int BN, int WM, int WN>
hipError_t tile_go(const MxLinear &p, int tiles, hipStream_t stream) {
    const int64_t mb = (p.rows + BM - 1) / BM, nb = (tiles + BN / 16 - 1) / (BN / 16);
    if (mb * nb > 0xfffff0) return hipErrorInvalidConfiguration;      // a launch has at most 2^32 - 1 threads
    hipLaunchKernelGGL((mx_tile_kernel<X8, GATED, BM, BN, WM, WN>), dim3((unsigned)((mb * nb + 7) / 8 * 8)), dim3(64 * WM * WN), 0,
                       stream, p, (uint32_t)mb, (uint32_t)nb);
    return hipGetLastError();
}

// The variant of the few-row kernel: the smallest tiles that make at most one workgroup a CU.  Smaller ones leave a part of the
// CUs a second workgroup to wait for, and read the rows or the weights more often.  Kernels alone, recorded, the weights in the
// caches, us for bf16 / 8-bit rows:
//   192 rows, K 5632, N 2048: 4 tiles x 32 rows (192 workgroups) 11.7 / 9.7, 2 x 32 (384) 13.9 / 11.5
//   16 rows, K 5632, N 6144: 2 x 16 (192) 5.7 / 5.5, 1 x 16 (384) 6.7 / 6.2; as fp32 15.7, 26.6
//   48 rows, K 5632, N 2048: 2 x 16 (192) 5.5 / 5.3, 1 x 16 (384) 6.4 / 6.0
// and one a CU against half of them: 64 rows, K 5632, N 2048: 2 x 16 (256) 5.9 / 5.5, 2 x 32 (128) 8.0 / 7.0; 32 rows, K 2048,
// N 8192: 2 x 32 (256) 5.3 / 4.8, 4 x 32 (128) 6.8 / 6.2.  It costs short sums a
// little: 192 rows, K 1024, N 2048: 5.3 / 5.0 against 6.1 / 4.9; one row, K 2048, N 12288: 5.1 / 4.4 against 4.8 / 4.2.
// The kernel for few rows up to where 4 x 32 makes one workgroup a CU: it has the whole sum in flight (128 rows, K 5632,
// N 2048: 8.7 / 7.4, 64 x 64 tiles 24.4 / 15.5).  Past that it has four waves, so that two are on a CU (64 rows, K 2048, gated
// 11264: 9.7 / 8.8, eight waves 12.8 / 10.5), and bf16 rows, whose tiles convert the weights in each of many steps one
// behind the other, keep it the longer the sum is.  Few / tiles, at N 8192 and gated 8192:
//   two a CU (128 rows): K 512 5.1 / 4.8 and 5.3 / 5.0, K 1024 7.0 / 6.9 and 7.2 / 7.1, K 2048 10.1 / 10.9 and 10.1 / 11.2
//   three (192 rows): K 1536 12.3 / 10.7 and 12.2 / 12.1, K 2048 14.1 / 13.0 and 14.2 / 15.2, K 5632 28.4 / 30.5 and 26.9 / 35.9
//   four (256 rows): K 2048 17.1 / 13.3 and 16.8 / 15.4, K 5632 34.1 / 31.3 and 33.9 / 36.4
// 8-bit rows: two a CU, K 2048 8.6 / 8.3 and 9.2 / 8.3, K 5632 17.2 / 19.0 and 17.1 / 23.4; with the weights from memory the few-row
// kernel is ahead throughout (9.9 / 14.4 and 10.3 / 14.5, 20.3 / 32.8 and 20.8 / 33.1).
// Tiles: largest with 5 workgroups for 4 CUs.  512 rows, K 2048, N 8192: 64 x 128 (512) 21.9 / 12.0, 64 x 64 (1,024) 23.7 /
// 18.5; 256 rows: 64 x 64 (512) 13.4 / 10.2, 64 x 128 (256) 14.5 / 9.8, from memory 15.1 / 14.8 and 15.7 / 15.6; 8-bit rows,
// N 32768, 512 rows: 128 x 256 (512) 33.5, 64 x 256 34.7, 256 rows: 64 x 256 (512) 19.2, 128 x 256 (256) 22.5.
// Rows that the kernel for few rows converts itself (MX_RAW_ROWS at most) stay as they are: fp32 or fp16, or of a width that
// ends inside a tile: one launch instead of two.  Past it, planes first / as they are, fp16 rows, kernels alone: 64 rows, K 2048,
// N 8192 12.6 / 13.4, N 2048 7.6 / 6.3, N 32000 26.1 / 51.7, gated 11264 16.6 / 19.0; 48 rows, K 5632, N 2048 14.5 / 18.9.
template <int X, bool GATED>
hipError_t mx_linear_t(const MxLinear &p, hipStream_t stream) {
    constexpr bool X8 = X == MX8;
    // the output's padding to whole 128s of columns counts as tiles (8-bit outputs: 8 pairs a 128)
    const int tiles = GATED && p.out == MX8 ? (p.N + 127) / 128 * 16 : p.T;
    const int64_t cus = device_cu_count();
    auto few = [&](int mt, int nb) { return (int64_t)((tiles + mt - 1) / mt) * ((p.rows + 16 * nb - 1) / (16 * nb)); };
    if constexpr (X == 0 || X == 2 || X == BF16_TAIL) {
        if constexpr (!GATED) {
            if (few(1, 1) <= cus) return few_rows_go<X, GATED, 1, 1, 8>(p, tiles, stream);
            if (few(2, 1) <= cus) return few_rows_go<X, GATED, 2, 1, 8>(p, tiles, stream);
        }
        return few_rows_go<X, GATED, 4, 1, 8>(p, tiles, stream);
    } else {
        const int sum = p.C * p.planes, most = X8 || sum <= 6 ? 1 : sum <= (GATED ? 12 : 16) ? 2 : 3;
        if (p.rows <= MX_RAW_ROWS || few(4, 2) <= most * cus) {
            if constexpr (!GATED) {
                if (few(1, 1) <= cus) return few_rows_go<X, GATED, 1, 1, 8>(p, tiles, stream);
                if (few(2, 1) <= cus) return few_rows_go<X, GATED, 2, 1, 8>(p, tiles, stream);
                if (p.rows > 16 && few(2, 2) <= cus) return few_rows_go<X, GATED, 2, 2, 8>(p, tiles, stream);
            }
            if (p.rows <= 16 || few(4, 1) <= cus) return few_rows_go<X, GATED, 4, 1, 8>(p, tiles, stream);
            if (few(4, 2) <= cus) return few_rows_go<X, GATED, 4, 2, 8>(p, tiles, stream);
            return few_rows_go<X, GATED, 4, 2, 4>(p, tiles, stream);
        }
        auto fills = [&](int bm, int bn) { return 4 * ((p.rows + bm - 1) / bm) * ((tiles + bn / 16 - 1) / (bn / 16)) >= 5 * cus; };
        if constexpr (X8)
            if (fills(128, 256)) return tile_go<X8, GATED, 128, 256, 2, 2>(p, tiles, stream);
        if (fills(64, 256)) return tile_go<X8, GATED, 64, 256, 1, 4>(p, tiles, stream);
        if (fills(64, 128)) return tile_go<X8, GATED, 64, 128, 2, 2>(p, tiles, stream);
        // a gated block of 32 columns takes four tiles of a wave
        if constexpr (GATED) return tile_go<X8, GATED, 64, 64, 4, 1>(p, tiles, stream);
        else return tile_go<X8, GATED, 64, 64, 2, 2>(p, tiles, stream);
    }
}

}  // namespace

hipError_t mx_linear(const MxLinear &p, hipStream_t stream) {
    if (p.x_type == MX8) return p.gated ? mx_linear_t<MX8, true>(p, stream) : mx_linear_t<MX8, false>(p, stream);
    if (p.x_type == 0) return p.gated ? mx_linear_t<0, true>(p, stream) : mx_linear_t<0, false>(p, stream);
    if (p.x_type == 2) return p.gated ? mx_linear_t<2, true>(p, stream) : mx_linear_t<2, false>(p, stream);
    if (p.K % 128) return p.gated ? mx_linear_t<BF16_TAIL, true>(p, stream) : mx_linear_t<BF16_TAIL, false>(p, stream);
    return p.gated ? mx_linear_t<1, true>(p, stream) : mx_linear_t<1, false>(p, stream);
}

}  // namespace vgdr
