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

__device__ __forceinline__ f32x2 buffer_load_nt2(__amdgpu_buffer_rsrc_t r, uint32_t voff) {
    return __builtin_bit_cast(f32x2, __builtin_amdgcn_raw_buffer_load_b64(r, (int)voff, 0, CPOL_NT));
}
__device__ __forceinline__ void buffer_store_nt2(f32x2 x, __amdgpu_buffer_rsrc_t r, uint32_t voff) {
    __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, x), r, (int)voff, 0, CPOL_NT);
}

// Two neighbouring channels of this (stream, head)'s q, k or v through the short conv: the cache moves
// to the a-th pending input, the block's inputs become pending, and put(t, x0, x1) takes the
// activated values.  TAPS: 4, all loads in flight at once; 0: any number up to 8, one token
// after the other (right-aligned in 8 places).
template <typename E, int LT, int TAPS, typename F>
__device__ __forceinline__ void draft_conv(const DraftParams &p, const E *src, int64_t ld, int64_t n, int a, int which, int col,
                                           F put) {
    constexpr int T = TAPS ? TAPS : 8;
    const int K = TAPS ? TAPS : p.cv.K, skip = T - K;
    const int64_t D = (int64_t)p.H * (which < 2 ? p.dk : p.dv);
    E *cache = reinterpret_cast<E *>(which == 0 ? p.cv.cq : which == 1 ? p.cv.ck : p.cv.cv) + n * K * D + col;
    E *pend = reinterpret_cast<E *>(which == 0 ? p.xq : which == 1 ? p.xk : p.xv) + n * p.P * D + col;
    const void *wp = which == 0 ? p.cv.wq : which == 1 ? p.cv.wk : p.cv.wv;
    const int wt = p.cv.w_f32 ? 0 : p.dtype;
    constexpr int NEW = TAPS ? LT : 1;
    Pair<E> x[T + NEW];                                            // the K last inputs, then the block's
    f32x2 w[T];
    unroll<T>([&](auto r) {
        x[r] = Pair<E>{(E)0.f, (E)0.f};
        w[r] = f32x2{0.f, 0.f};
        if (TAPS || r >= skip) {
            const int at = a + r - skip;                           // of the K cached and P pending inputs
            x[r] = *reinterpret_cast<const Pair<E> *>(at < K ? cache + at * D : pend + (at - K) * D);
            w[r] = f32x2{param_f(wp, wt, (int64_t)col * K + r - skip), param_f(wp, wt, (int64_t)(col + 1) * K + r - skip)};
        }
    });
    if (TAPS && p.L > 0)
        unroll<NEW>([&](auto t) { x[T + t] = *reinterpret_cast<const Pair<E> *>(src + (t < p.L ? (int)t : p.L - 1) * ld); });
    unroll<T>([&](auto r) {
        if (TAPS || r >= skip) *reinterpret_cast<Pair<E> *>(cache + (r - skip) * D) = x[r];
    });
    auto token = [&](int t, auto at) {                             // at: the token's place behind the window in x
        *reinterpret_cast<Pair<E> *>(pend + t * D) = x[T + at];
        f32x2 y = {0.f, 0.f};
        unroll<T>([&](auto r) {
            if (TAPS || r >= skip) {
                y[0] += w[r][0] * (float)x[at + 1 + r][0];
                y[1] += w[r][1] * (float)x[at + 1 + r][1];
            }
        });
        put(t, y[0] / (1.f + expf(-y[0])), y[1] / (1.f + expf(-y[1])));
    };
    if (TAPS) {
        unroll<NEW>([&](auto t) {
            if (t < p.L) token(t, t);
        });
    } else {
#pragma nounroll
        for (int t = 0; t < p.L; ++t) {
            x[T] = *reinterpret_cast<const Pair<E> *>(src + t * ld);
            token(t, std::integral_constant<int, 0>{});
            unroll<T>([&](auto r) { x[r] = x[r + 1]; });
        }
    }
}

}  // namespace

// One workgroup per (stream, head), a wave per 32 columns of the state, which it holds in the
// C layout of 16 x 16 tiles: lane 16 g + r has rows 16 i + 4 g + j (j < 4) of columns 2 r, 2 r + 1, so a
// row's 32 columns are one 128-byte line. As it lies it is the B operand of the product with [K; Q].
// RT: row tiles (dk <= 16 RT). LT: room of the pending block and tokens (8 or 16).
template <typename E, int GATE, int RT, int LT, int NT>
__global__ void __launch_bounds__(NT) __attribute__((amdgpu_waves_per_eu(LT == 16 && NT == 256 ? 3 : 4))) draft_block_kernel(const DraftParams p) {
    constexpr int DKP = 16 * RT, LDK = DKP + 4, WLD = DKP + 16, DVM = NT / 2, LP = DKP / 16;
    constexpr int SHARED = LT * WLD > 2 * LT * DVM ? LT * WLD : 2 * LT * DVM;
    __shared__ __attribute__((aligned(16))) float kk[LT][LDK], qq[LT][LDK], vv[LT][DVM];
    __shared__ __attribute__((aligned(16))) float both[SHARED];   // ws, then the products with the state
    __shared__ __attribute__((aligned(16))) float es[GATE == 2 ? LT : 1][GATE == 2 ? DKP : LT], ds[DKP];
    __shared__ __attribute__((aligned(16))) float aa[LT][LT], bb[LT][LT], betas[LT], decay[LT];
    const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 63, waves = nt >> 6;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), g4 = lane >> 4, r16 = lane & 15;
    const int64_t n = blockIdx.x / p.H;
    const int h = blockIdx.x - (int)n * p.H;
    const int dk = p.dk, dv = p.dv, L = p.L, P = p.P, pairs = dk + dv / 2;
    int a = p.accepted[n];
    a = a < 0 ? 0 : a > P ? P : a;

    // the state; rows and columns beyond it read zeros and are not stored
    const int col = 32 * wave + 2 * r16;
    const __amdgpu_buffer_rsrc_t rs = buffer_rsrc(p.S + (int64_t)blockIdx.x * dk * dv, (uint32_t)(dk * dv) * 4u);
    const uint32_t v0 = col < dv ? (uint32_t)(4 * g4 * dv + col) * 4u : 0x40000000u, row = (uint32_t)dv * 4u;
    f32x4 S[RT][2];
    unroll<RT>([&](auto i) {
        unroll<4>([&](auto j) {
            const f32x2 x = buffer_load_nt2(rs, v0 + (16 * i + j) * row);
            S[i][0][j.value] = x[0];
            S[i][1][j.value] = x[1];
        });
    });
    // the pending writes as the commit's B operand: token 4 s + g, this lane's columns
    f32x2 pu[LT / 4];
    unroll<LT / 4>([&](auto s) {
        const int t = 4 * s + g4;
        pu[s] = f32x2{0.f, 0.f};
        if (t < a && col < dv) pu[s] = *reinterpret_cast<const f32x2 *>(p.pu + ((n * P + t) * p.H + h) * dv + col);
    });
    // the accepted writes' weights at their block's end, a channel to a thread
    float *ws = both;
    const bool has_g = GATE == 2 || p.pg != nullptr;
    if (tid < DKP) {
        float pk[LT], pg[LT], run = 1.f;
        unroll<LT>([&](auto t) {
            const int64_t at = (n * P + t) * p.H + h;
            pk[t] = pg[t] = 0.f;
            if (t < a && tid < dk) {
                pk[t] = p.pk[at * dk + tid];
                if (has_g) pg[t] = p.pg[GATE == 2 ? at * dk + tid : at];
            }
        });
        unroll<LT>([&](auto s) {
            constexpr int t = LT - 1 - s;
            ws[t * WLD + tid] = t < a ? run * pk[t] : 0.f;
            if (t < a) run *= expf(pg[t]);
        });
        ds[tid] = run;
    }
    for (int cp = tid; cp < pairs; cp += nt) {
        const int c2 = 2 * cp, which = c2 < dk ? 0 : c2 < 2 * dk ? 1 : 2;
        const int c = which == 0 ? c2 : which == 1 ? c2 - dk : c2 - 2 * dk, cc = h * (which < 2 ? dk : dv) + c;
        const int64_t ld_in = which < 2 ? p.ld_qk : p.ld_v;
        const E *src = reinterpret_cast<const E *>(which == 0 ? p.q : which == 1 ? p.k : p.v) + n * L * ld_in + cc;
        float *to = which == 0 ? &qq[0][c] : which == 1 ? &kk[0][c] : &vv[0][c];
        const int ld = which < 2 ? LDK : DVM;
        auto put = [&](int t, float x, float y) { *reinterpret_cast<f32x2 *>(to + t * ld) = f32x2{x, y}; };
        if (p.cv.K == 4) draft_conv<E, LT, 4>(p, src, ld_in, n, a, which, cc, put);
        else if (p.cv.K) draft_conv<E, LT, 0>(p, src, ld_in, n, a, which, cc, put);
        else
            for (int t = 0; t < L; ++t) {
                const Pair<E> x = *reinterpret_cast<const Pair<E> *>(src + t * ld_in);
                put(t, (float)x[0], (float)x[1]);
            }
    }
    if (dk < DKP)
        for (int c = dk + tid; c < DKP; c += nt)
            for (int t = 0; t < LT; ++t) {
                kk[t][c] = qq[t][c] = 0.f;
                if (GATE == 2) es[t][c] = 1.f;
            }
    lds_barrier();
    // q, k to unit length, the decays and beta; from here on the pending block is the new one's
    if (L > 0) {
        if (p.fz.qk_l2norm) {
            for (int r = wave; r < 2 * L; r += waves) {
                float *x = r < L ? qq[r] : kk[r - L];
                float s = 0.f;
                for (int c = lane; c < dk; c += 64) s += x[c] * x[c];
                s = rsqrtf(wave_sum64(s) + 1e-6f);
                for (int c = lane; c < dk; c += 64) x[c] *= s;
            }
        }
        if (GATE == 1 && tid < L) {
            float g = 0.f;
            if (has_g) {
                g = reinterpret_cast<const float *>(p.g)[(n * L + tid) * p.H + h];
                p.pg[(n * P + tid) * p.H + h] = g;
            }
            es[0][tid] = expf(g);
        }
        if (GATE == 2) {
            for (int i = tid; i < L * dk; i += nt) {
                const int t = i / dk, c = i - t * dk;
                const int64_t at = ((n * L + t) * p.H + h) * dk + c;
                float g = p.fz.gate_16 ? (float)reinterpret_cast<const E *>(p.g)[at] : reinterpret_cast<const float *>(p.g)[at];
                if (p.fz.gate_act) {
                    const float z = g + p.fz.dt_bias[h * dk + c], al = expf(p.fz.A_log[h]);
                    g = p.fz.lb_set ? p.fz.lb / (1.f + expf(-al * z)) : -al * (z > 20.f ? z : log1pf(expf(z)));
                }
                p.pg[((n * P + t) * p.H + h) * dk + c] = g;
                es[t][c] = expf(g);
            }
        }
        if (tid < L) {
            const float b = p.use_delta ? p.beta[(n * L + tid) * p.H + h] : 0.f;
            betas[tid] = p.fz.beta_sigmoid ? 1.f / (1.f + expf(-b)) : b;
        }
        lds_barrier();
        for (int i = tid; i < L * dk; i += nt) {
            const int t = i / dk, c = i - t * dk;
            p.pk[((n * P + t) * p.H + h) * dk + c] = kk[t][c];
        }
        // A and B: 16 lanes share the channels of key j, decayed from token to token
        for (int j = tid >> 4; j < L; j += nt >> 4) {
            float x[LP];
#pragma unroll
            for (int c = 0; c < LP; ++c) x[c] = kk[j][r16 * LP + c];
            for (int t = j; t < L; ++t) {
                float sa = 0.f, sb = 0.f;
#pragma unroll
                for (int c = 0; c < LP; ++c) {
                    if (t > j) x[c] *= es[GATE == 2 ? t : 0][GATE == 2 ? r16 * LP + c : t];
                    sa += kk[t][r16 * LP + c] * x[c];
                    sb += qq[t][r16 * LP + c] * x[c];
                }
                sa = row_sum16(sa);
                sb = row_sum16(sb);
                if (r16 == 0) {
                    aa[t][j] = sa;
                    bb[t][j] = sb;
                }
            }
        }
        if (GATE == 2) {
            lds_barrier();
            for (int c = tid; c < dk; c += nt) {
                float run = 1.f;
                for (int t = 0; t < L; ++t) {
                    run *= es[t][c];
                    kk[t][c] *= run;
                    qq[t][c] *= run;
                }
            }
        } else if (tid == 0) {
            float run = 1.f;
            for (int t = 0; t < L; ++t) {
                run *= es[0][t];
                decay[t] = run;
            }
        }
        lds_barrier();
    }

    // commit
    unroll<RT>([&](auto i) {
        const f32x4 d = ld4(&ds[16 * i + 4 * g4]);
        S[i][0] *= d;
        S[i][1] *= d;
        unroll<LT / 4>([&](auto s) {
            const float w = ws[(4 * s + g4) * WLD + 16 * i + r16];
            S[i][0] = __builtin_amdgcn_mfma_f32_16x16x4f32(w, pu[s][0], S[i][0], 0, 0, 0);
            S[i][1] = __builtin_amdgcn_mfma_f32_16x16x4f32(w, pu[s][1], S[i][1], 0, 0, 0);
        });
    });
    uint32_t v1 = v0;
    asm volatile("" : "+v"(v1));                                   // the loads' 32 addresses are not kept for the stores
    unroll<RT>([&](auto i) {
        unroll<4>([&](auto j) { buffer_store_nt2(f32x2{S[i][0][j.value], S[i][1][j.value]}, rs, v1 + (16 * i + j) * row); });
    });
    if (L == 0) return;

    // [K; Q] S: rows 0 .. LT - 1 are K's, LT .. 2 LT - 1 Q's
    f32x4 z[LT / 8][2];
    unroll<LT / 8>([&](auto m) { z[m][0] = z[m][1] = f32x4{0.f, 0.f, 0.f, 0.f}; });
    unroll<RT>([&](auto i) {
        unroll<LT / 8>([&](auto m) {
            const float *x = LT == 16 ? (m ? qq[r16] : kk[r16]) : (r16 < 8 ? kk[r16 & 7] : qq[r16 & 7]);
            const f32x4 f = ld4(x + 16 * i + 4 * g4);
            z[m][0] = mfma_kb1(f, S[i][0], z[m][0]);
            z[m][1] = mfma_kb1(f, S[i][1], z[m][1]);
        });
    });
    lds_barrier();                                                 // ws is read no more
    float *prod = both;
    unroll<LT / 8>([&](auto m) {
        unroll<4>([&](auto j) {
            *reinterpret_cast<f32x2 *>(&prod[(16 * m + 4 * g4 + j) * DVM + col]) = f32x2{z[m][0][j.value], z[m][1][j.value]};
        });
    });
    lds_barrier();
    // the block's writes and outputs, a column to a lane (both halves of the wave the same)
    {
        const int c = 32 * wave + (lane & 31);
        float u[LT];
        unroll<LT>([&](auto t) {
            u[t] = 0.f;
            if (t < L) {
                float s = prod[t * DVM + c];
                if (GATE == 1) s *= decay[t];
                unroll<t>([&](auto j) { s += aa[t][j] * u[j]; });
                u[t] = p.use_delta ? betas[t] * (vv[t][c] - s) : vv[t][c];
                if (lane < 32 && c < dv) p.pu[((n * P + t) * p.H + h) * dv + c] = u[t];
                float o = prod[(LT + t) * DVM + c];
                if (GATE == 1) o *= decay[t];
                unroll<t + 1>([&](auto j) { o += bb[t][j] * u[j]; });
                if (lane < 32) vv[t][c] = p.scale * o;
            }
        });
    }
    lds_barrier();
    // the outputs, a wave per token
    for (int t = wave; t < L; t += waves) {
        E *out = reinterpret_cast<E *>(p.o) + ((n * L + t) * p.H + h) * dv;
        const E *gate = reinterpret_cast<const E *>(p.ep.gate) + (n * L + t) * p.ld_v + h * dv;
        float r = 1.f;
        if (p.ep.gate) {
            float s = 0.f;
            for (int c = lane; c < dv; c += 64) s += vv[t][c] * vv[t][c];
            r = rsqrtf(wave_sum64(s) / (float)dv + p.ep.eps);
        }
        for (int c = 2 * lane; c < dv; c += 128) {
            f32x2 x = *reinterpret_cast<const f32x2 *>(&vv[t][c]);
            if (p.ep.gate) {
                const Pair<E> z = *reinterpret_cast<const Pair<E> *>(gate + c);
#pragma unroll
                for (int b = 0; b < 2; ++b)
                    x[b] = x[b] * r * param_f(p.ep.gamma, p.ep.gamma_f32 ? 0 : p.dtype, c + b) *
                           ((float)z[b] / (1.f + expf(-(float)z[b])));
            }
            *reinterpret_cast<Pair<E> *>(out + c) = Pair<E>{(E)x[0], (E)x[1]};
        }
    }
}

template <typename E, int GATE, int RT, int LT>
static hipError_t draft_launch(const DraftParams &p, hipStream_t stream) {
    // a wave per 32 columns, and a thread per key channel
    const int by_cols = (p.dv + 31) / 32, waves = by_cols > RT / 4 ? by_cols : RT / 4;
    const dim3 grid((unsigned)(p.N * p.H)), block(64 * waves);
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
