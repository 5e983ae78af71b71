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
#include "gdr_common.hpp"
#include "gdr_kernels.hpp"

namespace vgdr {

namespace {

constexpr int DRAFT_L = DRAFT_MAX;

template <typename E> __device__ __forceinline__ float gate_in(const DraftParams &p, int64_t i) {
    return p.fz.gate_16 ? (float)reinterpret_cast<const E *>(p.g)[i] : reinterpret_cast<const float *>(p.g)[i];
}

// Channel c (0 .. 2 dk + dv - 1: q, k, then v) of this (stream, head)'s short conv: the
// cache moves to the a-th pending input, the new block's inputs become pending, and
// put(t, x) takes the activated values.
template <typename E, typename F>
__device__ __forceinline__ void draft_conv_channel(const DraftParams &p, int64_t n, int h, int a, int c, F put) {
    const int which = c < p.dk ? 0 : c < 2 * p.dk ? 1 : 2;
    const int d = which < 2 ? p.dk : p.dv;
    const int col = h * d + (which == 0 ? c : which == 1 ? c - p.dk : c - 2 * p.dk);
    const int64_t D = (int64_t)p.H * d;
    const E *raw = reinterpret_cast<const E *>(which == 0 ? p.q : which == 1 ? p.k : p.v) +
                   n * p.L * (which < 2 ? p.ld_qk : p.ld_v) + col;
    const int64_t ld = which < 2 ? p.ld_qk : p.ld_v;
    const int K = p.cv.K;
    if (K == 0) {
        for (int t = 0; t < p.L; ++t) put(t, (float)raw[t * ld]);
        return;
    }
    E *cache = reinterpret_cast<E *>(which == 0 ? p.cv.cq : which == 1 ? p.cv.ck : p.cv.cv) + n * K * D + col;
    E *pend = reinterpret_cast<E *>(which == 0 ? p.xq : which == 1 ? p.xk : p.xv) + n * p.P * D + col;
    const void *wp = which == 0 ? p.cv.wq : which == 1 ? p.cv.wk : p.cv.wv;
    float x[8], w[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) {
        E e = (E)0.f;
        if (r < K) e = a + r < K ? cache[(a + r) * D] : pend[(a + r - K) * D];
        x[r] = (float)e;
        w[r] = r < K ? param_f(wp, p.cv.w_f32 ? 0 : (sizeof(E) == 4 ? 0 : p.dtype), (int64_t)col * K + r) : 0.f;
    }
#pragma unroll
    for (int r = 0; r < 8; ++r)
        if (r < K) cache[r * D] = (E)x[r];
    for (int t = 0; t < p.L; ++t) {
        const E e = raw[t * ld];
        pend[t * D] = e;
        float y = 0.f;
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            if (r + 1 < K) x[r] = x[r + 1];
            else if (r + 1 == K) x[r] = (float)e;
            y += r < K ? w[r] * x[r] : 0.f;
        }
        put(t, y / (1.f + expf(-y)));
    }
}

}  // namespace

// One workgroup per (stream, head), a thread per column of the state, which it walks
// token by token in registers.
template <typename E, int GATE, int DKP>
__global__ void __launch_bounds__(256) draft_walk_kernel(const DraftParams p) {
    __shared__ float qs[DRAFT_L][DKP], ks[DRAFT_L][DKP], es[DRAFT_L][GATE == 2 ? DKP : 1], vs[DRAFT_L][256];
    __shared__ float ws[DRAFT_L][DKP], ds[DKP], bs[DRAFT_L];
    const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 63, wave = tid >> 6, waves = nt >> 6;
    const int64_t n = blockIdx.x / p.H;
    const int h = blockIdx.x - (int)n * p.H;
    const int dk = p.dk, dv = p.dv, L = p.L, P = p.P;
    int a = p.accepted[n];
    a = a < 0 ? 0 : a > P ? P : a;
    // what the accepted writes weigh at the end of the block they came in
    for (int c = tid; c < DKP; c += nt) {
        float run = 1.f;
        for (int t = a - 1; t >= 0; --t) {
            const int64_t at = (n * P + t) * p.H + h;
            ws[t][c] = c < dk ? run * p.pk[at * dk + c] : 0.f;
            if (GATE == 1) run *= expf(p.pg[at]);
            if (GATE == 2 && c < dk) run *= expf(p.pg[at * dk + c]);
        }
        ds[c] = run;
    }
    __syncthreads();
    float S[DKP];
    float *state = p.S + (int64_t)blockIdx.x * dk * dv + tid;
    if (tid < dv) {
#pragma unroll
        for (int i = 0; i < DKP; ++i) S[i] = i < dk ? ds[i] * state[i * dv] : 0.f;
        for (int t = 0; t < a; ++t) {
            const float u = p.pu[((n * P + t) * p.H + h) * dv + tid];
#pragma unroll
            for (int i = 0; i < DKP; ++i) S[i] += ws[t][i] * u;
        }
#pragma unroll
        for (int i = 0; i < DKP; ++i)
            if (i < dk) state[i * dv] = S[i];
    }
    // the new block's q, k, v; past here the pending block is the new one's
    __syncthreads();
    for (int c = tid; c < 2 * dk + dv; c += nt) {
        float *to = c < dk ? &qs[0][c] : c < 2 * dk ? &ks[0][c - dk] : &vs[0][c - 2 * dk];
        const int ld = c < 2 * dk ? DKP : 256;
        draft_conv_channel<E>(p, n, h, a, c, [&](int t, float x) { to[t * ld] = x; });
    }
    if (L == 0) return;
    for (int c = dk + tid; c < DKP; c += nt)
        for (int t = 0; t < L; ++t) qs[t][c] = ks[t][c] = 0.f;
    __syncthreads();
    if (p.fz.qk_l2norm) {
        for (int r = wave; r < 2 * L; r += waves) {
            float *x = r < L ? qs[r] : ks[r - L];
            float s = 0.f;
            for (int c = lane; c < dk; c += 64) s += x[c] * x[c];
            s = rsqrtf(wave_sum64(s) + 1e-6f);
            for (int c = lane; c < dk; c += 64) x[c] *= s;
        }
    }
    if (GATE == 1 && tid < L) {
        const int64_t at = (n * L + tid) * p.H + h;
        const float g = gate_in<float>(p, at);
        p.pg[(n * P + tid) * p.H + h] = g;
        es[tid][0] = expf(g);
    }
    if (GATE == 2) {
        for (int i = tid; i < L * DKP; i += nt) {
            const int t = i / DKP, c = i - t * DKP;
            if (c >= dk) {
                es[t][c] = 1.f;
                continue;
            }
            float g = gate_in<E>(p, ((n * L + t) * p.H + h) * dk + c);
            if (p.fz.gate_act) {
                const float z = g + p.fz.dt_bias[h * dk + c], al = expf(p.fz.A_log[h]);
                g = p.fz.lb_set ? p.fz.lb / (1.f + expf(-al * z)) : -al * (z > 20.f ? z : log1pf(expf(z)));
            }
            p.pg[((n * P + t) * p.H + h) * dk + c] = g;
            es[t][c] = expf(g);
        }
    }
    if (p.use_delta && tid < L) {
        const float b = p.beta[(n * L + tid) * p.H + h];
        bs[tid] = p.fz.beta_sigmoid ? 1.f / (1.f + expf(-b)) : b;
    }
    __syncthreads();
    for (int i = tid; i < L * dk; i += nt) {
        const int t = i / dk, c = i - t * dk;
        p.pk[((n * P + t) * p.H + h) * dk + c] = ks[t][c];
    }
    if (tid < dv) {
        for (int t = 0; t < L; ++t) {
            float kS = 0.f, o = 0.f;
#pragma unroll
            for (int i = 0; i < DKP; ++i) {
                if (GATE) S[i] *= es[t][GATE == 2 ? i : 0];
                kS += ks[t][i] * S[i];
            }
            const float u = p.use_delta ? bs[t] * (vs[t][tid] - kS) : vs[t][tid];
#pragma unroll
            for (int i = 0; i < DKP; ++i) {
                S[i] += ks[t][i] * u;
                o += qs[t][i] * S[i];
            }
            p.pu[((n * P + t) * p.H + h) * dv + tid] = u;
            vs[t][tid] = p.scale * o;
        }
    }
    __syncthreads();
    // the outputs, a wave per token
    for (int t = wave; t < L; t += waves) {
        E *out = reinterpret_cast<E *>(p.o) + ((n * L + t) * p.H + h) * dv;
        float r = 1.f;
        if (p.ep.gate) {
            float s = 0.f;
            for (int c = lane; c < dv; c += 64) s += vs[t][c] * vs[t][c];
            r = rsqrtf(wave_sum64(s) / (float)dv + p.ep.eps);
        }
        const E *gate = reinterpret_cast<const E *>(p.ep.gate) + (n * L + t) * p.ld_v + h * dv;
        for (int c = lane; c < dv; c += 64) {
            float x = vs[t][c];
            if (p.ep.gate) {
                const float z = (float)gate[c];
                x = x * r * param_f(p.ep.gamma, p.ep.gamma_f32 ? 0 : p.dtype, c) * (z / (1.f + expf(-z)));
            }
            out[c] = (E)x;
        }
    }
}

template <typename E, int GATE>
static hipError_t draft_launch(const DraftParams &p, hipStream_t stream) {
    const dim3 grid((unsigned)(p.N * p.H)), block(64 * ((p.dv + 63) / 64));
    if (p.dk <= 64) draft_walk_kernel<E, GATE, 64><<<grid, block, 0, stream>>>(p);
    else draft_walk_kernel<E, GATE, 128><<<grid, block, 0, stream>>>(p);
    return hipGetLastError();
}

template <typename E>
static hipError_t draft_typed(int gate, const DraftParams &p, hipStream_t stream) {
    return gate == 0 ? draft_launch<E, 0>(p, stream) : gate == 1 ? draft_launch<E, 1>(p, stream) : draft_launch<E, 2>(p, stream);
}

hipError_t draft_step(int gate, const DraftParams &p, hipStream_t stream) {
    if (p.dtype == 0) return draft_typed<float>(gate, p, stream);
    if (p.dtype == 1) return draft_typed<__bf16>(gate, p, stream);
    return draft_typed<_Float16>(gate, p, stream);
}

}  // namespace vgdr
