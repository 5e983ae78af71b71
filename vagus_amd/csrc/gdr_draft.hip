// One step of speculative decoding through a gated delta-rule layer, from the
// projections of a block of drafted tokens to the input of W_o (draft_step), for
// every (stream, head) with its state S in R^{dk x dv}:
//
//  * commit: of the last block's tokens the first a = accepted[stream] stand. Their
//    writes, kept since then as k_t, u_t and the log-decay g_t, join the state:
//        S <- diag(e^{g_1 + .. + g_a}) S + sum_{t <= a} diag(e^{g_{t+1} + .. + g_a}) k_t u_t^T
//    and the conv caches move to the a-th of the block's raw inputs. A write u_t does not
//    depend on the tokens behind it, so those that fall leave no trace.
//  * block: the producers of the layer's decode step (short conv + SiLU behind the
//    cache, q, k L2 norm, gate activation, beta sigmoid) over L <= 16 new tokens, then
//        S' <- diag(e^{g_t}) S';  u_t = beta_t (v_t - S'^T k_t);  S' <- S' + k_t u_t^T;
//        o_t = scale S'^T q_t
//    on a copy S' of the state, and the output epilogue; k_t, u_t, g_t and the raw inputs
//    stay behind as the next call's pending block. The state itself is not moved.
//
// Everything between the inputs and the outputs is fp32: unlike the one-token decode step
// no intermediate is rounded to the element type.
//
// The block is not walked: with G_t the running log-decay, A_tj = k_t . e^{G_t - G_j} k_j and
// B_tj = q_t . e^{G_t - G_j} k_j,
//     u_t = beta_t (v_t - S^T e^{G_t} k_t - sum_{j < t} A_tj u_j)
//     o_t = scale (S^T e^{G_t} q_t + sum_{j <= t} B_tj u_j)
// which touches the state in one product of [K; Q] with S (fp32 MFMA) for the whole block.
// The decays between two tokens are products of the tokens' own, never a difference of two
// running sums, so a strong one loses nothing.
#include "gdr_common.hpp"
#include "gdr_kernels.hpp"

namespace vgdr {

namespace {

template <typename E> using Pair = E __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float buffer_load1(__amdgpu_buffer_rsrc_t r, uint32_t voff) {
    return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(r, (int)voff, 0, 0));
}
__device__ __forceinline__ f32x2 buffer_load2(__amdgpu_buffer_rsrc_t r, uint32_t voff) {
    return __builtin_bit_cast(f32x2, __builtin_amdgcn_raw_buffer_load_b64(r, (int)voff, 0, 0));
}
__device__ __forceinline__ f32x4 buffer_load4(__amdgpu_buffer_rsrc_t r, uint32_t voff) {
    return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)voff, 0, 0));
}
constexpr uint32_t NOWHERE = 0x40000000u;                          // an offset behind every block: reads zeros

// by value: a choice among a parameter block's members would put the block into scratch memory
__device__ __forceinline__ uint64_t pick(int which, const void *q, const void *k, const void *v) {
    const uint64_t a = (uint64_t)q, b = (uint64_t)k, c = (uint64_t)v;
    return which == 0 ? a : which == 1 ? b : c;
}

// Two neighbouring channels of this (stream, head)'s q, k or v: where they are.
template <typename E> struct ChannelPair {
    const E *src;                 // the block's inputs, ld apart
    E *cache, *pend;              // the conv's last K inputs and the pending block's, D apart
    const void *w;                // the conv's weights of the two
    int64_t ld, D;
    int which, c;                 // 0 q, 1 k, 2 v; channel in the head

    __device__ __forceinline__ ChannelPair(const DraftParams &p, int64_t n, int h, int cp) {
        const int c2 = 2 * cp, K = p.cv.K;
        which = c2 < p.dk ? 0 : c2 < 2 * p.dk ? 1 : 2;
        c = which == 0 ? c2 : which == 1 ? c2 - p.dk : c2 - 2 * p.dk;
        const int d = which < 2 ? p.dk : p.dv, col = h * d + c;
        ld = which < 2 ? p.ld_qk : p.ld_v;
        D = (int64_t)p.H * d;
        src = reinterpret_cast<const E *>(pick(which, p.q, p.k, p.v)) + n * p.L * ld + col;
        cache = reinterpret_cast<E *>(pick(which, p.cv.cq, p.cv.ck, p.cv.cv)) + n * K * D + col;
        pend = reinterpret_cast<E *>(pick(which, p.xq, p.xk, p.xv)) + n * p.P * D + col;
        w = reinterpret_cast<const char *>(pick(which, p.cv.wq, p.cv.wk, p.cv.wv)) + (int64_t)col * K * (p.cv.w_f32 ? 4 : (int)sizeof(E));
    }
};

// The short conv of any number of taps up to 8, one token after the other: the cache moves to the
// a-th pending input, the block's inputs become pending, put(t, x0, x1) takes the activated values.
template <typename E, typename F>
__device__ __forceinline__ void draft_conv_any(const DraftParams &p, const ChannelPair<E> &at, int a, F put) {
    const int K = p.cv.K, skip = 8 - K, wt = p.cv.w_f32 ? 0 : p.dtype;
    Pair<E> x[9];                                                  // right-aligned: the K last inputs, then a token's
    f32x2 w[8];
    unroll<8>([&](auto r) {
        x[r] = Pair<E>{(E)0.f, (E)0.f};
        w[r] = f32x2{0.f, 0.f};
        if (r >= skip) {
            const int i = a + r - skip;                            // of the K cached and P pending inputs
            x[r] = *reinterpret_cast<const Pair<E> *>(i < K ? at.cache + i * at.D : at.pend + (i - K) * at.D);
            w[r] = f32x2{param_f(at.w, wt, r - skip), param_f(at.w, wt, K + r - skip)};
        }
    });
    unroll<8>([&](auto r) {
        if (r >= skip) *reinterpret_cast<Pair<E> *>(at.cache + (r - skip) * at.D) = x[r];
    });
#pragma nounroll
    for (int t = 0; t < p.L; ++t) {
        x[8] = *reinterpret_cast<const Pair<E> *>(at.src + t * at.ld);
        *reinterpret_cast<Pair<E> *>(at.pend + t * at.D) = x[8];
        f32x2 y = {0.f, 0.f};
        unroll<8>([&](auto r) {
            if (r >= skip) {
                y[0] += w[r][0] * (float)x[1 + r][0];
                y[1] += w[r][1] * (float)x[1 + r][1];
            }
        });
        put(t, y[0] * sigmoidf_(y[0]), y[1] * sigmoidf_(y[1]));
        unroll<8>([&](auto r) { x[r] = x[r + 1]; });
    }
}

// inclusive sums over the lanes behind, within a row of 16
__device__ __forceinline__ float row_suffix16(float x) {
    x += dpp_f<0x101>(x);                                          // row_shl:1
    x += dpp_f<0x102>(x);
    x += dpp_f<0x104>(x);
    x += dpp_f<0x108>(x);
    return x;
}
__device__ __forceinline__ float row_prefix16(float x) {
    x += dpp_f<0x111>(x);                                          // row_shr:1
    x += dpp_f<0x112>(x);
    x += dpp_f<0x114>(x);
    x += dpp_f<0x118>(x);
    return x;
}

}  // namespace

// One workgroup per (stream, head). A wave holds 64 rows x 64 columns of the state in the C layout of
// 16 x 16 tiles: lane 16 g + r has rows 16 i + 4 g + j (i, j < 4) of columns 4 r .. 4 r + 3, so that an
// access touches four rows of 256 bytes (32 columns a wave, 128 bytes a row: a bare copy of the state
// took 42 us where this takes 26). As it lies it is the B operand of the product with [K; Q], whose
// two halves of rows (dk > 64) meet in LDS.  q and k are kept unnormalised: the norms are A's and
// q's own diagonals and scale the results.  RT: row tiles (dk <= 16 RT). LT: room of the pending
// block and tokens: 16, or 8, whose [K; Q] is one tile of 16 rows and which, without per-channel gates, leaves
// registers and LDS for four workgroups a CU (three at 16).  Per-channel gates of dk > 64 take 147 registers a
// thread at 8 tokens (three waves a SIMD) and at 16 and dv <= 128 283 with 70 KB of LDS: one wave a SIMD, since pk, pg
// and the operands in flight live beside the state across A and B. At 8 tokens the per-channel kernels of dk <= 64 and
// the fp32 ones of other gates keep 5 to 17 registers in scratch memory (7 in fp32 at 16 and dv <= 128).  At least 128 (RT 4) or 256 threads,
// two per value channel, and one per pair of q, k, v channels.
//
// Bound by the state's way in and out: 64 streams of 16 128 x 128 heads, bf16, blocks of 5: 28 us for 161 MB
// (5.7 TB/s) on one state again and again, which the last-level cache holds in part, 29-30 (5.4) on eight in turn;
// 160 MB pass behind the L2. The products and the solve, which the stores cover in part, are 5 of it;
// 128 streams, blocks of 16: 93-97 us for 411 MB (99 on several in turn), where the product with the state costs
// 9, the solve 13 and the outputs 6. One workgroup a CU (64 streams of 4 128 x 256 heads, per-channel
// gates, blocks of 8) is a chain of latencies: 25 us for 83 MB. One stream: 10 us.  Per-channel gates on
// the first case's heads: 41 us for 166 MB, 106 for 222 MB at 16 tokens (54 without), where A and B, walked a key at a
// time, and the one wave a SIMD show. The commit alone (L = 0): 23.5 us, per-channel 26.4.
// Measured and left out: the operands' loads ahead of the state's (b64 31.1 -> 33.1 us), stores before
// the products (32.6) or behind the solve (32.9), ws and the products in one LDS area for a fourth
// workgroup at 16 tokens (97 -> 135 us with the registers that takes).
template <typename E, int GATE, int RT, int LT, int NT>
__global__ void __launch_bounds__(NT) __attribute__((amdgpu_waves_per_eu(GATE == 2 && RT == 8 ? (NT == 256 ? 3 : 2) : LT == 8 ? 4 : NT == 256 ? 3 : 2)))
draft_block_kernel(const DraftParams p) {
    constexpr int DKP = 16 * RT, LDK = DKP + 4, WLD = DKP + 16, DVM = NT / 2, NC = DKP / 64, HALVES = RT / 4, LG = LT / 4;
    __shared__ __attribute__((aligned(16))) float kk[LT][LDK], qq[LT][LDK], vv[LT][DVM], ws[LT][WLD], prod[2 * LT][DVM];
    __shared__ __attribute__((aligned(16))) float es[GATE == 2 ? LT : 1][GATE == 2 ? DKP : 16];  // e^{g_t}
    __shared__ __attribute__((aligned(16))) float eg[GATE == 2 ? LT : 1][GATE == 2 ? LDK : 16];  // e^{G_t}
    __shared__ __attribute__((aligned(16))) float ds[GATE == 2 ? DKP : 16], aa[LT][LT], bb[LT][LT];
    __shared__ float betas[16], rk[LT], rq[LT], squares[NT / 128][LT];
    const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 63, waves = nt >> 6;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), g4 = lane >> 4, r16 = lane & 15;
    const int64_t n = blockIdx.x / p.H;
    const int h = blockIdx.x - (int)n * p.H;
    const int dk = p.dk, dv = p.dv, L = p.L, P = p.P, H = p.H, pairs = dk + dv / 2;
    int a = p.accepted[n];
    // --- the state; rows and columns beyond it read zeros and are not stored ---
    const int half = wave % HALVES, col = 64 * (wave / HALVES) + 4 * r16;
    const __amdgpu_buffer_rsrc_t rs = buffer_rsrc(p.S + (int64_t)blockIdx.x * dk * dv, (uint32_t)(dk * dv) * 4u);
    const uint32_t row = (uint32_t)dv * 4u, v0 = col < dv ? (uint32_t)((64 * half + 4 * g4) * dv + col) * 4u : NOWHERE;
    f32x4 S[4][4];                                                 // [row tile][column of the lane's four]
    unroll<4>([&](auto i) {
        unroll<4>([&](auto j) {
            const f32x4 y = buffer_load_nt4(rs, v0 + (16 * i + j) * row, 0);
            unroll<4>([&](auto c) { S[i][c][j.value] = y[c.value]; });
        });
    });

    // --- without the state ---
    a = a < 0 ? 0 : a > P ? P : a;
    // scalar gate and beta: lane r of every row of 16 has token r's
    const bool has_g = GATE == 2 || p.pg != nullptr;
    const uint32_t lane_h = (uint32_t)(r16 * H + h) * 4u;
    const float be = buffer_load1(buffer_rsrc(p.use_delta ? p.beta + n * L * H : nullptr, p.use_delta ? (uint32_t)(L * H) * 4u : 0u), lane_h);
    float gp = 0.f, gn = 0.f;
    f32x2 gv[GATE == 2 ? LG : 1], dt_bias[GATE == 2 ? LG : 1];     // per channel: two channels of some tokens
    if (GATE == 1) {
        gp = buffer_load1(buffer_rsrc(p.pg + (has_g ? n * P * H : 0), has_g ? (uint32_t)(P * H) * 4u : 0u), r16 < a ? lane_h : NOWHERE);
        const uint32_t e = p.fz.gate_16 ? 2 : 4;
        const __amdgpu_buffer_rsrc_t bg = buffer_rsrc(reinterpret_cast<const char *>(p.g) + (has_g ? n * L * H * e : 0),
                                                      has_g ? (uint32_t)(L * H) * e : 0u);
        if constexpr (sizeof(E) == 2) {
            if (p.fz.gate_16) gn = (float)__builtin_bit_cast(E, __builtin_amdgcn_raw_buffer_load_b16(bg, (int)(lane_h / 2), 0, 0));
            else gn = buffer_load1(bg, lane_h);
        } else {
            gn = buffer_load1(bg, lane_h);
        }
    }
    if (GATE == 2) {
        const uint32_t e = p.fz.gate_16 ? 2 : 4;
        const __amdgpu_buffer_rsrc_t bg = buffer_rsrc(reinterpret_cast<const char *>(p.g) + n * L * H * dk * e, (uint32_t)(L * H * dk) * e);
        const __amdgpu_buffer_rsrc_t bb_ = buffer_rsrc(p.fz.dt_bias, p.fz.gate_act ? (uint32_t)(H * dk) * 4u : 0u);
        unroll<LG>([&](auto m) {
            const int i = tid + m * nt, t = i / (DKP / 2), c = 2 * (i % (DKP / 2));
            const uint32_t o = t < L && c < dk ? (uint32_t)((t * H + h) * dk + c) * e : NOWHERE;
            f32x2 &g = gv[GATE == 2 ? m : 0];
            if (p.fz.gate_16) g[0] = buffer_load1(bg, o);          // both halves
            else g = buffer_load2(bg, o);
            dt_bias[GATE == 2 ? m : 0] = buffer_load2(bb_, c < dk ? (uint32_t)(h * dk + c) * 4u : NOWHERE);
        });
    }
    // the short conv, a thread to two channels
    {
        const ChannelPair<E> at(p, n, h, tid < pairs ? tid : pairs - 1);
        float *to = at.which == 0 ? &qq[0][at.c] : at.which == 1 ? &kk[0][at.c] : &vv[0][at.c];
        const int ld = at.which < 2 ? LDK : DVM;
        auto put = [&](int t, float y0, float y1) { *reinterpret_cast<f32x2 *>(to + t * ld) = f32x2{y0, y1}; };
        if (p.conv4) {
            Pair<E> x[4 + LT];                                     // the last inputs, then the block's
            u32x4 wraw[2];
            const bool w32 = sizeof(E) == 4 || p.cv.w_f32;
            unroll<4>([&](auto r) {
                const int i = a + r;
                x[r] = *reinterpret_cast<const Pair<E> *>(i < 4 ? at.cache + i * at.D : at.pend + (i - 4) * at.D);
            });
            wraw[0] = *reinterpret_cast<const u32x4 *>(at.w);
            wraw[1] = reinterpret_cast<const u32x4 *>(at.w)[w32 ? 1 : 0];
            if (L > 0)
                unroll<LT>([&](auto t) { x[4 + t] = *reinterpret_cast<const Pair<E> *>(at.src + (t < L ? (int)t : L - 1) * at.ld); });
            f32x2 w[4];
            unroll<8>([&](auto i) {
                const unsigned word = w32 ? wraw[i / 4][i % 4] : wraw[0][i / 2];
                float f = __builtin_bit_cast(float, word);
                if constexpr (sizeof(E) == 2)
                    if (!w32) f = (float)__builtin_bit_cast(E, (unsigned short)(i % 2 ? word >> 16 : word));
                w[i % 4][i / 4] = f;
            });
            if (tid < pairs) {
                unroll<4>([&](auto r) { *reinterpret_cast<Pair<E> *>(at.cache + r * at.D) = x[r]; });
                unroll<LT>([&](auto t) {
                    if (t < L) {
                        *reinterpret_cast<Pair<E> *>(at.pend + t * at.D) = x[4 + t];
                        f32x2 y = {0.f, 0.f};
                        unroll<4>([&](auto r) {
                            y[0] += w[r][0] * (float)x[t + 1 + r][0];
                            y[1] += w[r][1] * (float)x[t + 1 + r][1];
                        });
                        put(t, y[0] * sigmoidf_(y[0]), y[1] * sigmoidf_(y[1]));
                    }
                });
            }
        } else if (tid < pairs) {
            if (p.cv.K) draft_conv_any<E>(p, at, a, put);
            else
                for (int t = 0; t < L; ++t) {
                    const Pair<E> y = *reinterpret_cast<const Pair<E> *>(at.src + t * at.ld);
                    put(t, (float)y[0], (float)y[1]);
                }
        }
    }
    // the pending keys (and per-channel decays), a channel to a thread, and writes, as the commit's B
    // operand: token 4 s + g, this lane's columns
    float pk[LT], pg[GATE == 2 ? LT : 1];
    f32x4 pu[LG];
    {
        const uint32_t kr = (uint32_t)(H * dk) * 4u, k0 = (uint32_t)(h * dk + tid) * 4u;
        const uint32_t ur = (uint32_t)(H * dv) * 4u, u0 = (uint32_t)(h * dv + col) * 4u;
        const __amdgpu_buffer_rsrc_t bk = buffer_rsrc(p.pk + n * P * H * dk, (uint32_t)P * kr);
        const __amdgpu_buffer_rsrc_t bu = buffer_rsrc(p.pu + n * P * H * dv, (uint32_t)P * ur);
        unroll<LT>([&](auto t) { pk[t] = buffer_load1(bk, t < a && tid < dk ? k0 + t * kr : NOWHERE); });
        if (GATE == 2) {
            const __amdgpu_buffer_rsrc_t bg = buffer_rsrc(p.pg + n * P * H * dk, (uint32_t)P * kr);
            unroll<LT>([&](auto t) { pg[GATE == 2 ? t : 0] = buffer_load1(bg, t < a && tid < dk ? k0 + t * kr : NOWHERE); });
        }
        unroll<LG>([&](auto s) {
            const int t = 4 * s + g4;
            pu[s] = buffer_load4(bu, t < a && col < dv ? u0 + t * ur : NOWHERE);
        });
    }
    if (GATE == 2) {
        const float al = p.fz.gate_act ? p.fz.A_log[h] : 0.f;
        unroll<LG>([&](auto m) {
            const int i = tid + m * nt, t = i / (DKP / 2), c = 2 * (i % (DKP / 2));
            f32x2 &g = gv[GATE == 2 ? m : 0], &b = dt_bias[GATE == 2 ? m : 0];
            if constexpr (sizeof(E) == 2)
                if (p.fz.gate_16) {
                    const Pair<E> x = __builtin_bit_cast(Pair<E>, g[0]);
                    g = f32x2{(float)x[0], (float)x[1]};
                }
            if (p.fz.gate_act) {
                g[0] = gate_activation(g[0], al, b[0], p.fz.lb_set, p.fz.lb);
                g[1] = gate_activation(g[1], al, b[1], p.fz.lb_set, p.fz.lb);
            }
            if (t < LT) *reinterpret_cast<f32x2 *>(&es[GATE == 2 ? t : 0][c]) = f32x2{__expf(g[0]), __expf(g[1])};
        });
    } else if (tid < 16) {
        if (p.fz.gate_act) gn = -__expf(p.fz.A_log[h]) * softplusf_(gn + p.fz.dt_bias[h]);
        es[0][tid] = __expf(gn);
        eg[0][tid] = __expf(row_prefix16(gn));
    }
    if (tid < 16) betas[tid] = p.fz.beta_sigmoid ? sigmoidf_(be) : be;
    if (dk < DKP)
        for (int c = dk + tid; c < DKP; c += nt)
            for (int t = 0; t < LT; ++t) kk[t][c] = qq[t][c] = 0.f;
    lds_barrier();
    // A and B
    if (GATE == 2) {
        // per channel: 16 lanes share the channels of key j, which decays from token to token
        for (int j = wave + waves * g4; j < L; j += 4 * waves) {
            f32x4 y[NC];
            unroll<NC>([&](auto c) { y[c] = ld4(&kk[j][64 * c + 4 * r16]); });
            for (int t = j; t < L; ++t) {
                float sa = 0.f, sb = 0.f, sq = 0.f;
                unroll<NC>([&](auto c) {
                    const f32x4 k4 = ld4(&kk[t][64 * c + 4 * r16]), q4 = ld4(&qq[t][64 * c + 4 * r16]);
                    if (t > j) y[c] *= ld4(&es[GATE == 2 ? t : 0][64 * c + 4 * r16]);
                    unroll<4>([&](auto i) {
                        sa += k4[i.value] * y[c][i.value];
                        sb += q4[i.value] * y[c][i.value];
                        sq += q4[i.value] * q4[i.value];
                    });
                });
                sa = row_sum16(sa);
                sb = row_sum16(sb);
                if (t == j) sq = row_sum16(sq);
                if (r16 == 0) {
                    aa[t][j] = sa;
                    bb[t][j] = sb;
                    if (t == j) {
                        rk[t] = p.fz.qk_l2norm ? rsqrtf(sa + 1e-6f) : 1.f;
                        rq[t] = p.scale * (p.fz.qk_l2norm ? rsqrtf(sq + 1e-6f) : 1.f);
                    }
                }
            }
        }
    } else {
        // [K; Q] K^T by MFMA, two tiles of channels to a wave, joined in LDS in a fixed order, and the tokens'
        // decays between (blocks of 16, 128 streams of 16 heads: 97 us with the loop above)
        constexpr int SHARES = RT / 2, TILES = LT / 8;
        float *shares = &prod[0][0];                               // [SHARES][TILES][16][16]
        if (wave < SHARES) {
            f32x4 y[TILES];
            unroll<TILES>([&](auto m) { y[m] = f32x4{0.f, 0.f, 0.f, 0.f}; });
            unroll<2>([&](auto s) {
                const int c = 16 * (2 * wave + s) + 4 * g4;
                const f32x4 k4 = ld4(&kk[r16 % LT][c]), q4 = ld4(&qq[r16 % LT][c]);
                if (LT == 8) {
                    y[0] = mfma_kb1(r16 < 8 ? k4 : q4, k4, y[0]);
                } else {
                    y[0] = mfma_kb1(k4, k4, y[0]);
                    y[TILES - 1] = mfma_kb1(q4, k4, y[TILES - 1]);
                }
            });
            unroll<TILES>([&](auto m) {
                unroll<4>([&](auto j) { shares[((wave * TILES + m) * 16 + 4 * g4 + j) * 16 + r16] = y[m][j.value]; });
            });
        }
        for (int t = wave; t < L; t += waves) {
            float s = 0.f;
            for (int c = lane; c < dk; c += 64) s += qq[t][c] * qq[t][c];
            s = wave_sum64(s);
            if (lane == 0) rq[t] = p.scale * (p.fz.qk_l2norm ? rsqrtf(s + 1e-6f) : 1.f);
        }
        lds_barrier();
        for (int i = tid; i < L * LT; i += nt) {
            const int t = i / LT, j = i % LT;
            if (j > t) continue;
            float sa = 0.f, sb = 0.f, run = 1.f;
            unroll<SHARES>([&](auto w) {
                sa += shares[(w * TILES * 16 + t) * 16 + j];
                sb += shares[(w * TILES * 16 + LT + t) * 16 + j];
            });
            for (int e = j + 1; e <= t; ++e) run *= es[0][e];
            aa[t][j] = run * sa;
            bb[t][j] = run * sb;
            if (j == t) rk[t] = p.fz.qk_l2norm ? rsqrtf(sa + 1e-6f) : 1.f;
        }
    }
    // what the accepted writes weigh at their block's end
    if (GATE == 2) {
        for (int c = tid; c < dk; c += nt) {
            float run = 1.f;
            for (int t = 0; t < L; ++t) {
                run *= es[GATE == 2 ? t : 0][c];
                eg[GATE == 2 ? t : 0][c] = run;
            }
        }
        if (dk < DKP)
            for (int c = dk + tid; c < DKP; c += nt)
                for (int t = 0; t < LT; ++t) eg[GATE == 2 ? t : 0][c] = 1.f;
        if (tid < DKP) {
            float run = 1.f;
            unroll<LT>([&](auto s) {
                constexpr int t = LT - 1 - s;
                ws[t][tid] = run * pk[t];
                run *= __expf(pg[GATE == 2 ? t : 0]);              // 1 behind the accepted
            });
            ds[GATE == 2 ? tid : 0] = run;
        }
    } else {
        if (tid < DKP) unroll<LT>([&](auto t) { ws[t][tid] = pk[t]; });
        const float back = row_suffix16(gp), weight = __expf(dpp_f<0x101>(back));
        unroll<LG>([&](auto s) { pu[s] *= __shfl(weight, 4 * s + g4); });
        if (tid < 16) ds[0] = __expf(__shfl(back, 0));
    }
    lds_barrier();
    // the pending block has been read: from here on it is the new one's
    if (GATE == 1 && has_g && tid < L) p.pg[(n * P + tid) * H + h] = gn;
    if (GATE == 2)
        unroll<LG>([&](auto m) {
            const int i = tid + m * nt, t = i / (DKP / 2), c = 2 * (i % (DKP / 2));
            if (t < L && c < dk) *reinterpret_cast<f32x2 *>(p.pg + ((n * P + t) * H + h) * dk + c) = gv[GATE == 2 ? m : 0];
        });
    for (int i = tid; i < L * (DKP / 2); i += nt) {
        const int t = i / (DKP / 2), c = 2 * (i % (DKP / 2));
        const f32x2 y = *reinterpret_cast<const f32x2 *>(&kk[t][c]);
        if (c < dk) *reinterpret_cast<f32x2 *>(p.pk + ((n * P + t) * H + h) * dk + c) = f32x2{y[0] * rk[t], y[1] * rk[t]};
    }

    // --- commit ---
    unroll<4>([&](auto i) {
        const int k0 = 64 * half + 16 * i;
        const f32x4 d = GATE == 2 ? ld4(&ds[GATE == 2 ? k0 + 4 * g4 : 0]) : f32x4{ds[0], ds[0], ds[0], ds[0]};
        unroll<4>([&](auto c) { S[i][c] *= d; });
        unroll<LG>([&](auto s) {
            const float w = ws[4 * s + g4][k0 + r16];
            unroll<4>([&](auto c) { S[i][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(w, pu[s][c.value], S[i][c], 0, 0, 0); });
        });
    });
    if (L == 0) {
    uint32_t v1 = v0;
    asm volatile("" : "+v"(v1));                                   // the loads' addresses are not kept for the stores
    unroll<4>([&](auto i) {
        unroll<4>([&](auto j) {
            buffer_store_nt4(f32x4{S[i][0][j.value], S[i][1][j.value], S[i][2][j.value], S[i][3][j.value]}, rs,
                             v1 + (16 * i + j) * row, 0);
        });
    });
        return;
    }

    // the output gate's rows and gamma, for the end
    const int half_dv = dv / 2;
    Pair<E> ogate[LG];
    f32x2 gamma[LG];
    unroll<LG>([&](auto m) {
        const int i = tid + m * nt, t = i / half_dv, c = 2 * (i - t * half_dv);
        ogate[m] = Pair<E>{(E)0.f, (E)0.f};
        gamma[m] = f32x2{0.f, 0.f};
        if (p.ep.gate && t < L) {
            ogate[m] = *reinterpret_cast<const Pair<E> *>(reinterpret_cast<const E *>(p.ep.gate) + (n * L + t) * p.ld_v + h * dv + c);
            if (p.ep.gamma_f32) {
                gamma[m] = reinterpret_cast<const f32x2 *>(p.ep.gamma)[c / 2];
            } else {
                const Pair<E> y = reinterpret_cast<const Pair<E> *>(p.ep.gamma)[c / 2];
                gamma[m] = f32x2{(float)y[0], (float)y[1]};
            }
        }
    });

    // --- [K; Q] S: rows 0 .. LT - 1 are K's, LT .. 2 LT - 1 Q's ---
    f32x4 z[LT / 8][4];
    unroll<LT / 8>([&](auto m) { unroll<4>([&](auto c) { z[m][c] = f32x4{0.f, 0.f, 0.f, 0.f}; }); });
    unroll<4>([&](auto i) {
        unroll<LT / 8>([&](auto m) {
            const int k0 = 64 * half + 16 * i + 4 * g4;
            f32x4 f = ld4(LT == 16 ? (m ? &qq[r16 % LT][k0] : &kk[r16 % LT][k0]) : (r16 < 8 ? &kk[r16 & 7][k0] : &qq[r16 & 7][k0]));
            if (GATE == 2) f *= ld4(&eg[GATE == 2 ? r16 % LT : 0][k0]);
            unroll<4>([&](auto c) { z[m][c] = mfma_kb1(f, S[i][c], z[m][c]); });
        });
    });
    uint32_t v1 = v0;
    asm volatile("" : "+v"(v1));                                   // the loads' addresses are not kept for the stores
    unroll<4>([&](auto i) {
        unroll<4>([&](auto j) {
            buffer_store_nt4(f32x4{S[i][0][j.value], S[i][1][j.value], S[i][2][j.value], S[i][3][j.value]}, rs,
                             v1 + (16 * i + j) * row, 0);
        });
    });
    const bool mine = col - 4 * r16 < dv;                          // a wave with columns
    auto exchange = [&](auto f) {
        unroll<LT / 8>([&](auto m) {
            unroll<4>([&](auto j) {
                f(*reinterpret_cast<f32x4 *>(&prod[16 * m + 4 * g4 + j][col]), m, j);
            });
        });
    };
    if (HALVES == 2) {
        if (mine && half == 1)
            exchange([&](f32x4 &x, auto m, auto j) { x = f32x4{z[m][0][j.value], z[m][1][j.value], z[m][2][j.value], z[m][3][j.value]}; });
        lds_barrier();
    }
    // the block's writes and outputs, a column to a lane
    if (mine && half == 0) {
        exchange([&](f32x4 &x, auto m, auto j) {
            const f32x4 y = {z[m][0][j.value], z[m][1][j.value], z[m][2][j.value], z[m][3][j.value]};
            x = HALVES == 2 ? x + y : y;
        });
        const int c = 64 * (wave / HALVES) + lane;
        float u[LT];                                               // rk_t u_t
        unroll<LT>([&](auto t) {
            u[t] = 0.f;
            if (t < L) {
                float s = prod[t][c], o = prod[LT + t][c], v = vv[t][c];
                const float k1 = rk[t];
                if (GATE == 1) {
                    s *= eg[0][t];
                    o *= eg[0][t];
                }
                unroll<t>([&](auto j) { s += aa[t][j] * u[j]; });
                if (p.use_delta) v = betas[t] * (v - k1 * s);
                if (c < dv) p.pu[((n * P + t) * H + h) * dv + c] = v;
                u[t] = k1 * v;
                unroll<t + 1>([&](auto j) { o += bb[t][j] * u[j]; });
                o *= rq[t];
                vv[t][c] = o;
                if (p.ep.gate) {
                    const float q = wave_sum64(c < dv ? o * o : 0.f);
                    if (lane == 0) squares[wave / HALVES][t] = q;
                }
            }
        });
    }
    lds_barrier();
    // --- the outputs, a thread to two columns of up to LG tokens ---
    unroll<LG>([&](auto m) {
        const int i = tid + m * nt, t = i / half_dv, c = 2 * (i - t * half_dv);
        if (t < L) {
            f32x2 y = *reinterpret_cast<const f32x2 *>(&vv[t][c]);
            if (p.ep.gate) {
                float s = squares[0][t];
                for (int b = 1; 64 * b < dv; ++b) s += squares[b][t];
                const float r = rsqrtf(s / (float)dv + p.ep.eps);
                y[0] *= r * gamma[m][0] * ((float)ogate[m][0] * sigmoidf_((float)ogate[m][0]));
                y[1] *= r * gamma[m][1] * ((float)ogate[m][1] * sigmoidf_((float)ogate[m][1]));
            }
            *reinterpret_cast<Pair<E> *>(reinterpret_cast<E *>(p.o) + ((n * L + t) * H + h) * dv + c) = Pair<E>{(E)y[0], (E)y[1]};
        }
    });
}

// a wave per 64 x 64 of the state, a thread per pair of q, k, v channels and per two key or value channels of
// LT / 4 tokens
int64_t draft_threads(int64_t dk, int64_t dv) {
    const int64_t rt = dk <= 64 ? 4 : 8, tiles = rt / 4 * ((dv + 63) / 64), pairs = (dk + dv / 2 + 63) / 64, least = (dv + 31) / 32;
    int64_t waves = tiles > pairs ? tiles : pairs;
    waves = waves > least ? waves : least;
    return 64 * (waves > rt / 2 ? waves : rt / 2);
}

template <typename E, int GATE, int RT, int LT>
static hipError_t draft_launch(const DraftParams &p, hipStream_t stream) {
    const dim3 grid((unsigned)(p.N * p.H)), block((unsigned)draft_threads(p.dk, p.dv));
    if (p.dv <= 128) draft_block_kernel<E, GATE, RT, LT, 256><<<grid, block, 0, stream>>>(p);
    else draft_block_kernel<E, GATE, RT, LT, 512><<<grid, block, 0, stream>>>(p);
    return hipGetLastError();
}

template <typename E, int GATE>
static hipError_t draft_sized(const DraftParams &p, hipStream_t stream) {
    if (p.dk <= 64) return p.P <= 8 ? draft_launch<E, GATE, 4, 8>(p, stream) : draft_launch<E, GATE, 4, 16>(p, stream);
    return p.P <= 8 ? draft_launch<E, GATE, 8, 8>(p, stream) : draft_launch<E, GATE, 8, 16>(p, stream);
}

template <typename E>
static hipError_t draft_typed(int gate, const DraftParams &p, hipStream_t stream) {
    return gate == 2 ? draft_sized<E, 2>(p, stream) : draft_sized<E, 1>(p, stream);
}

hipError_t draft_step(int gate, const DraftParams &p, hipStream_t stream) {
    if (p.dtype == 0) return draft_typed<float>(gate, p, stream);
    if (p.dtype == 1) return draft_typed<__bf16>(gate, p, stream);
    return draft_typed<_Float16>(gate, p, stream);
}

}  // namespace vgdr
