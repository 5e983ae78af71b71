// What a speculative decoding step does beside the layers, for every stream:
//
//  * verify_drafts: which of K drafted tokens stand before the target's logits, and
//    the token that follows them (row_mass_kernel, choose_kernel).
//  * lookup_drafts: the next step's drafts, from the stream's own text (lookup_kernel).
#include "gdr_common.hpp"
#include "gdr_kernels.hpp"

namespace vgdr {

namespace {

constexpr int ROW_THREADS = 256;

// A logit as it counts: NaN never has any mass
template <typename E> __device__ __forceinline__ float logit(E x) {
    const float f = (float)x;
    return f == f ? f : -__builtin_inff();
}

// e^{(x - top) / T} in 64 bits; the top itself is 1 whatever its value, infinities and a row of nothing
// but -inf included
__device__ __forceinline__ double mass(float x, float top, double inv_t) {
    return x == top ? 1.0 : exp(((double)x - (double)top) * inv_t);
}

__device__ __forceinline__ double prob_f(const void *q, int dtype, int64_t i) { return (double)param_f(q, dtype, i); }

}  // namespace

// Per (stream, position): the row's top, the lowest index that has it, and (T > 0) its
// whole mass sum_v e^{(x_v - top) / T}.
template <typename E>
__global__ void __launch_bounds__(ROW_THREADS) row_mass_kernel(const VerifyParams p) {
    __shared__ float tops[ROW_THREADS];
    __shared__ int ats[ROW_THREADS];
    __shared__ double sums[ROW_THREADS];
    const int tid = threadIdx.x;
    const int64_t n = blockIdx.x / (p.K + 1), i = blockIdx.x - n * (p.K + 1);
    const E *x = reinterpret_cast<const E *>(p.logits) + n * p.ld_stream + i * p.ld_row;
    float top = -__builtin_inff();
    int at = p.V;
    for (int v = tid; v < p.V; v += ROW_THREADS) {
        const float f = logit(x[v]);
        if (f > top || at == p.V) {
            top = f;
            at = v;
        }
    }
    tops[tid] = top;
    ats[tid] = at;
    __syncthreads();
    for (int j = 0; j < ROW_THREADS; ++j)
        if (tops[j] > top || (tops[j] == top && ats[j] < at)) {
            top = tops[j];
            at = ats[j];
        }
    const double t = (double)p.temperature[n];
    double s = 0.0;
    if (t > 0.0)
        for (int v = tid; v < p.V; v += ROW_THREADS) s += mass(logit(x[v]), top, 1.0 / t);
    sums[tid] = s;
    __syncthreads();
    if (tid == 0) {
        s = 0.0;
        for (int j = 0; j < ROW_THREADS; ++j) s += sums[j];
        p.rows[blockIdx.x] = RowMass{s, top, at};
    }
}

// Per stream: the drafts that stand and the token behind them.
template <typename E>
__global__ void __launch_bounds__(ROW_THREADS) choose_kernel(const VerifyParams p) {
    __shared__ double sums[ROW_THREADS];
    __shared__ int chosen;
    const int tid = threadIdx.x, K = p.K, V = p.V;
    const int64_t n = blockIdx.x;
    const double t = (double)p.temperature[n], inv_t = 1.0 / t;
    const float *u = p.uniforms + n * (K + 1);
    const RowMass *rows = p.rows + n * (K + 1);
    int n_drafts = p.n_drafts ? p.n_drafts[n] : K;
    n_drafts = n_drafts < 0 ? 0 : n_drafts > K ? K : n_drafts;
    int i = 0;
    for (; i < n_drafts; ++i) {
        const int64_t d = p.drafts[n * K + i];
        if (d < 0 || d >= V) break;                                        // no such token
        const E *x = reinterpret_cast<const E *>(p.logits) + n * p.ld_stream + i * p.ld_row;
        const double q = p.probs ? prob_f(p.probs, p.probs_dtype, n * p.ld_probs_stream + i * p.ld_probs_row + d) : 1.0;
        const double w = t > 0.0 ? mass(logit(x[d]), rows[i].top, inv_t) : (d == rows[i].at ? 1.0 : 0.0);
        const double z = t > 0.0 ? rows[i].sum : 1.0;
        if (!((double)u[i] * q * z < w)) break;
    }
    int token = rows[i].at;
    if (t > 0.0) {
        // the row's mass, or where a draft was refused what it has more than the draft's: by slices of the row
        const E *x = reinterpret_cast<const E *>(p.logits) + n * p.ld_stream + i * p.ld_row;
        const float top = rows[i].top;
        const double z = rows[i].sum;
        const int64_t d = i < n_drafts ? p.drafts[n * K + i] : -1;
        const int64_t qrow = n * p.ld_probs_stream + i * p.ld_probs_row;
        const int per = (V + ROW_THREADS - 1) / ROW_THREADS, v0 = tid * per, v1 = v0 + per < V ? v0 + per : V;
        for (int residual = i < n_drafts ? 1 : 0; residual >= 0; --residual) {
            auto left = [&](int v) {
                const double w = mass(logit(x[v]), top, inv_t);
                if (!residual) return w;
                if (!p.probs) return v == d ? 0.0 : w;
                const double r = w - z * prob_f(p.probs, p.probs_dtype, qrow + v);
                return r > 0.0 ? r : 0.0;
            };
            double s = 0.0;
            for (int v = v0; v < v1; ++v) s += left(v);
            __syncthreads();
            sums[tid] = s;
            __syncthreads();
            double whole = 0.0;
            for (int j = 0; j < ROW_THREADS; ++j) whole += sums[j];
            if (!(whole > 0.0)) continue;                                  // the draft's probabilities cover the row's
            if (tid == 0) {
                const double goal = (double)u[K] * whole;
                double c = 0.0;
                int j = 0, last = 0;
                for (; j < ROW_THREADS; ++j) {
                    if (sums[j] > 0.0) last = j;
                    if (c + sums[j] > goal) break;
                    c += sums[j];
                }
                if (j == ROW_THREADS) {
                    j = last;
                    c -= sums[last];
                }
                int found = -1;
                for (int v = j * per; v < (j + 1) * per && v < V; ++v) {
                    const double w = left(v);
                    if (w > 0.0) found = v;
                    c += w;
                    if (c > goal && w > 0.0) break;
                }
                chosen = found < 0 ? rows[i].at : found;
            }
            __syncthreads();
            token = chosen;
            break;
        }
    }
    for (int j = tid; j <= K; j += ROW_THREADS)
        p.tokens[n * (K + 1) + j] = j < i ? p.drafts[n * K + j] : j == i ? token : -1;
    if (tid == 0) p.accepted[n] = i;
}

hipError_t verify_drafts(int dtype, const VerifyParams &p, hipStream_t stream) {
    const dim3 rows((unsigned)(p.N * (p.K + 1))), streams((unsigned)p.N), block(ROW_THREADS);
    if (dtype == 0) {
        row_mass_kernel<float><<<rows, block, 0, stream>>>(p);
        choose_kernel<float><<<streams, block, 0, stream>>>(p);
    } else if (dtype == 1) {
        row_mass_kernel<__bf16><<<rows, block, 0, stream>>>(p);
        choose_kernel<__bf16><<<streams, block, 0, stream>>>(p);
    } else {
        row_mass_kernel<_Float16><<<rows, block, 0, stream>>>(p);
        choose_kernel<_Float16><<<streams, block, 0, stream>>>(p);
    }
    return hipGetLastError();
}

int64_t verify_workspace(int64_t N, int64_t K, int64_t V) { return N * (K + 1) * (int64_t)sizeof(RowMass); }

// Per stream: of all places e < n - 1 of its n tokens at which at least `shortest` of the last
// tokens end as well, the one where most of them do (up to `longest`), of those the last; the
// drafts are what follows it, again from there where the text ends.
template <typename I>
__global__ void __launch_bounds__(ROW_THREADS) lookup_kernel(const LookupParams p) {
    __shared__ long long keys[ROW_THREADS];
    const int tid = threadIdx.x;
    const int64_t b = blockIdx.x;
    const I *text = reinterpret_cast<const I *>(p.history) + b * p.ld;
    int64_t n = p.lengths[b];
    n = n < 0 ? 0 : n > p.cap ? p.cap : n;
    long long best = -1;
    for (int64_t e = tid; e < n - 1; e += ROW_THREADS) {
        int m = 0;
        while (m < p.longest && m <= e && text[e - m] == text[n - 1 - m]) ++m;
        const long long key = ((long long)m << 40) | e;
        if (m >= p.shortest && key > best) best = key;
    }
    keys[tid] = best;
    __syncthreads();
    for (int j = 0; j < ROW_THREADS; ++j) best = keys[j] > best ? keys[j] : best;
    const int64_t start = (best & ((1LL << 40) - 1)) + 1;
    for (int64_t i = tid; i < p.K; i += ROW_THREADS)
        p.drafts[b * p.K + i] = best < 0 ? 0 : (int64_t)text[start + i % (n - start)];
    if (tid == 0) p.counts[b] = best < 0 ? 0 : p.K;
}

hipError_t lookup_drafts(bool wide, const LookupParams &p, hipStream_t stream) {
    if (wide) lookup_kernel<int64_t><<<dim3((unsigned)p.N), dim3(ROW_THREADS), 0, stream>>>(p);
    else lookup_kernel<int32_t><<<dim3((unsigned)p.N), dim3(ROW_THREADS), 0, stream>>>(p);
    return hipGetLastError();
}

}  // namespace vgdr
