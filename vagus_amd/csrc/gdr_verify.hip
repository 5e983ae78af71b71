// What a speculative decoding step does beside the layers, for every stream:
//
//  * verify_drafts: which of K drafted tokens stand before the target's logits, and
//    the token that follows them.  row_mass_kernel reads every row once, each wave a chunk of 2048
//    logits held in registers: its top, and where it is (greedy streams) or sum e^{(x - top) / T}
//    in fp32, which decides u q Z < w but where the two are within 1e-5.  stand_kernel decides, and
//    of the one row that a stream samples sums the weights in 64 bits, in blocks of 512 over several
//    workgroups: the running sums meet the uniform number at up to V borders, so an fp32
//    sum's error (5e-7) would choose another token once in some ten streams of 100,000 ids, the
//    64-bit weights' (2e-13, their exponential's) never in practice.  rest_kernel does the same with what the draft's probabilities
//    leave of the row, and choose_kernel finds the token.  The last workgroup of a stream to finish
//    does not do it: the fence that takes writes the L2 back (58 us a call at 64 streams of 32,000
//    ids); nor does one workgroup do all: 26 us with the weights on 64 of 256 CUs.
//  * lookup_drafts: the next step's drafts, from the stream's own text (lookup_kernel).
#include "gdr_common.hpp"
#include "gdr_kernels.hpp"

namespace vgdr {

namespace {

constexpr int CHUNK = 2048, BLOCK = 512, EACH = BLOCK / 64;        // logits of a wave in row_mass, in the others; a lane's
constexpr int ROW_WAVES = 4, WAVES = 8;                            // of a workgroup: in row_mass, in the others
constexpr int64_t SHARE = 512;
constexpr double LOG2E = 1.4426950408889634;

// A row in pieces on 16-byte boundaries: it starts at place `first` of the first.
template <typename E> struct Row {
    static constexpr int UNIT = 16 / (int)sizeof(E);
    const E *base;
    int first;
    int64_t end;                                                   // first + V
    __device__ __forceinline__ Row(const void *x, int V) {
        const uint64_t a = (uint64_t)x;
        base = reinterpret_cast<const E *>(a & ~15ull);
        first = (int)(a & 15) / (int)sizeof(E);
        end = (int64_t)first + V;
    }
    // N logits of a lane from place `from` (of 64 N) in order of their place: x[UNIT k + e] is place 64 UNIT k
    // + UNIT lane + e behind it (place()).  What is not the row's is -inf; NaN stays.
    template <int N> __device__ __forceinline__ void load(int64_t from, int lane, float (&x)[N]) const {
        constexpr int UNITS = N / UNIT;
        const int64_t left = end - from;
        const uint32_t bytes = (uint32_t)((left < 64 * N ? (left > 0 ? left : 0) : 64 * N) * sizeof(E));
        const __amdgpu_buffer_rsrc_t r = buffer_rsrc(base + from, (bytes + 15) & ~15u);  // the last unit whole
        u32x4 raw[UNITS];
        unroll<UNITS>([&](auto k) {
            raw[k] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (64 * k + lane) * 16, 0, 0));
        });
        unroll<UNITS>([&](auto k) {
            typedef E V16 __attribute__((ext_vector_type(UNIT)));
            const V16 v = __builtin_bit_cast(V16, raw[k]);
            unroll<UNIT>([&](auto e) { x[UNIT * k + e] = (float)v[e.value]; });
        });
        if (left < 64 * N || from < first)
            unroll<N>([&](auto i) {
                if (!has(from + place(i, lane))) x[i] = -__builtin_inff();
            });
    }
    __device__ static __forceinline__ int place(int i, int lane) { return 64 * UNIT * (i / UNIT) + UNIT * lane + i % UNIT; }
    __device__ __forceinline__ bool has(int64_t a) const { return a >= first && a < end; }
};

__device__ __forceinline__ float wave_max(float x) {
    for (int m = 32; m; m >>= 1) x = fmaxf(x, __shfl_xor(x, m));
    return x;
}
__device__ __forceinline__ int wave_min(int x) {
    for (int m = 32; m; m >>= 1) {
        const int y = __shfl_xor(x, m);
        x = y < x ? y : x;
    }
    return x;
}
// DPP as dpp_f, both halves
template <int CTRL, int ROW_MASK = 0xf>
__device__ __forceinline__ double dpp_d(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROW_MASK, 0xf, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, ROW_MASK, 0xf, false);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double lane_d(double x, int lane) {     // x of one lane, the same for all
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)u, lane), hi = __builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), lane);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// inclusive sums over the lanes up to this one (wave_scan in 64 bits)
__device__ __forceinline__ double wave_prefix(double x) {
    x += dpp_d<0x111>(x);
    x += dpp_d<0x112>(x);
    x += dpp_d<0x114>(x);
    x += dpp_d<0x118>(x);
    x += dpp_d<0x142, 0xa>(x);
    x += dpp_d<0x143, 0xc>(x);
    return x;
}
__device__ __forceinline__ double wave_sum(double x) { return lane_d(wave_prefix(x), 63); }
// the first lane whose running sum `upto` passes the goal with something of its own, else the last that has
// any, else -1; passed: whether it is the former
__device__ __forceinline__ int passing_lane(double own, double upto, double goal, bool &passed) {
    const uint64_t past = __ballot(own > 0.0 && upto > goal), any = __ballot(own > 0.0);
    passed = past != 0;
    return past ? __ffsll((unsigned long long)past) - 1 : any ? 63 - __clzll((long long)any) : -1;
}

// e^{(x - top) / T} in 64 bits for a finite top, c = log2(e) / T: 2^n 2^f, n whole, |f| <= 1/2, by the exponential
// series of f ln 2 up to its 10th power (2e-13 off). n is rounded off and added to the exponent as an
// integer: the 64-bit rounding, conversion and scaling instructions run at a fraction of an addition's rate.
// Nothing below 2^-1000 and for NaN.
__device__ __forceinline__ double mass_finite(float x, float top, double c) {
    constexpr double L1 = 0.6931471805599453, L2 = L1 * L1 / 2, L3 = L2 * L1 / 3, L4 = L3 * L1 / 4, L5 = L4 * L1 / 5,
                     L6 = L5 * L1 / 6, L7 = L6 * L1 / 7, L8 = L7 * L1 / 8, L9 = L8 * L1 / 9, L10 = L9 * L1 / 10;
    constexpr double ROUND = 6755399441055744.0;                   // 1.5 2^52: the sum's last bit is worth 1
    const double y = ((double)x - (double)top) * c;
    const double r = y + ROUND, f = y - (r - ROUND);
    double s = fma(L10, f, L9);
    s = fma(s, f, L8);
    s = fma(s, f, L7);
    s = fma(s, f, L6);
    s = fma(s, f, L5);
    s = fma(s, f, L4);
    s = fma(s, f, L3);
    s = fma(s, f, L2);
    s = fma(s, f, L1);
    s = fma(s, f, 1.0);
    const uint64_t u = __builtin_bit_cast(uint64_t, s);
    const uint32_t hi = (uint32_t)(u >> 32) + ((uint32_t)__builtin_bit_cast(uint64_t, r) << 20);
    s = __builtin_bit_cast(double, (uint64_t)hi << 32 | (uint32_t)u);
    return y >= -1000.0 ? s : 0.0;
}
// the same for any top: of an infinite one what equals it counts 1 (NaN as -inf), all else nothing
__device__ __forceinline__ bool infinite(float top) { return fabsf(top) == __builtin_inff(); }
__device__ __forceinline__ double mass(float x, float top, double c) {
    if (infinite(top)) return fmaxf(x, -__builtin_inff()) == top ? 1.0 : 0.0;
    return mass_finite(x, top, c);
}

}  // namespace

// Per (stream, position, chunk): the top, and for a greedy stream the lowest id that has it, for a sampled one
// sum e^{(x - top) / T}.  Some ten vector instructions a logit, so that it is bound by reading them: 128 x 8 rows
// of 131,072, 268 MB, in 40-46 us, 5.8-6.7 TB/s (74 us at twenty, with the id sought and NaN turned to -inf everywhere).
template <typename E>
__global__ void __launch_bounds__(64 * ROW_WAVES) row_mass_kernel(const VerifyParams p) {
    constexpr int PER = CHUNK / 64;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t chunk = (int64_t)blockIdx.x * ROW_WAVES + wave, from = chunk * CHUNK;
    const int64_t line = blockIdx.y + (int64_t)blockIdx.z * gridDim.y;
    if (line >= p.N * (p.K + 1) || chunk >= p.chunks) return;
    const int64_t n = line / (p.K + 1), i = line - n * (p.K + 1);
    const Row<E> row(reinterpret_cast<const E *>(p.logits) + n * p.ld_stream + i * p.ld_row, p.V);
    const float t = p.temperature[n];
    float x[PER];
    row.load(from, lane, x);
    float top = -__builtin_inff();
    unroll<PER>([&](auto j) { top = fmaxf(top, x[j]); });
    top = wave_max(top);
    const int64_t v0 = from > row.first ? from : row.first, v1 = from + CHUNK < row.end ? from + CHUNK : row.end;
    const int count = v1 > v0 ? (int)(v1 - v0) : 0;               // of the row's own here
    int at = (int)(v0 - row.first);
    float s = (float)count;                                        // all -inf or NaN: all alike
    if (top > -__builtin_inff()) {
        s = 0.f;
        if (t > 0.f) {
            const float c = (float)(LOG2E / (double)t);
            if (top < __builtin_inff()) unroll<PER>([&](auto j) { s += __builtin_amdgcn_exp2f((x[j] - top) * c); });
            s = wave_sum64(s);
            if (!(s == s) || top == __builtin_inff()) {            // NaN among them, or +inf
                s = 0.f;
                unroll<PER>([&](auto j) {
                    const float e = __builtin_amdgcn_exp2f((x[j] - top) * c);
                    s += x[j] == top ? 1.f : e == e ? e : 0.f;
                });
                s = wave_sum64(s);
            }
        } else {
            int low = 0x7fffffff;
            unroll<PER>([&](auto j) {
                constexpr int k = PER - 1 - j;
                if (x[k] == top) low = Row<E>::place(k, lane);
            });
            at = (int)(from + wave_min(low) - row.first);
        }
    }
    if (lane == 0) p.rows[line * p.chunks + chunk] = RowMass{s, top, count ? at : -1};
}

namespace {

// A stream's row whose token is sampled: p_v = weight / whole.
template <typename E> struct Sampled {
    Row<E> row;
    int V;
    float top;
    double c;
    int without;                  // an id without mass (a certain draft that was refused), or -1
    const void *q;                // the draft's probabilities of this row, of which z times each is taken off, or NULL
    int q_dtype;
    double z;

    // block b's logits EACH lane .. EACH lane + EACH - 1 as they lie, in whole units of 16 bytes of the row
    struct Raw { u32x4 u[EACH * sizeof(E) / 16]; };
    __device__ __forceinline__ Raw raw(int64_t b, int lane) const {
        Raw r;
        unroll<EACH * (int)sizeof(E) / 16>([&](auto k) {
            const int64_t at = b * BLOCK + EACH * lane + Row<E>::UNIT * k;
            r.u[k] = at < row.end ? *reinterpret_cast<const u32x4 *>(row.base + at) : u32x4{0, 0, 0, 0};
        });
        return r;
    }
    // their weights
    __device__ __forceinline__ void weigh(const Raw &r, int64_t b, int lane, double (&w)[EACH]) const {
        const int64_t at = b * BLOCK + EACH * lane;
        float x[EACH], qv[EACH];
        unroll<EACH>([&](auto e) {
            if constexpr (sizeof(E) == 2)
                x[e] = (float)__builtin_bit_cast(E, (unsigned short)(r.u[0][e / 2] >> (e % 2 * 16)));
            else x[e] = __builtin_bit_cast(float, (unsigned)r.u[e / 4][e % 4]);
        });
        const int v0 = (int)(at - row.first);
        unroll<EACH>([&](auto e) { qv[e] = 0.f; });
        if (q) {
            auto fetch = [&](auto *q0) __attribute__((always_inline)) {  // ids outside the row: its nearest end's
                unroll<EACH>([&](auto e) {
                    const int v = v0 + e;
                    qv[e] = (float)q0[v < 0 ? 0 : v < V ? v : V - 1];
                });
            };
            if (q_dtype == 0) fetch(reinterpret_cast<const float *>(q));
            else if (q_dtype == 1) fetch(reinterpret_cast<const __bf16 *>(q));
            else fetch(reinterpret_cast<const _Float16 *>(q));
        }
        if (infinite(top)) {
            unroll<EACH>([&](auto e) { w[e] = fmaxf(x[e], -__builtin_inff()) == top ? 1.0 : 0.0; });
        } else {
            unroll<EACH>([&](auto e) {
                w[e] = mass_finite(x[e], top, c);
                if (e % 4 == 3) __builtin_amdgcn_sched_barrier(0);
            });
        }
        if (q) unroll<EACH>([&](auto e) { w[e] = fmax(w[e] - z * (double)qv[e], 0.0); });
        unroll<EACH>([&](auto e) {
            const int v = v0 + e;
            if (v < 0 || v >= V || v == without) w[e] = 0.0;
        });
    }
    __device__ __forceinline__ static double sum(const double (&w)[EACH]) {
        double s = 0.0;
        unroll<EACH>([&](auto e) { s += w[e]; });
        return s;
    }
    // f(b, sum of its weights) for the blocks b = first, first + step, ..; a block's logits are loaded two ahead
    template <typename F> __device__ __forceinline__ void sums(int64_t first, int64_t step, int64_t blocks, int lane, F f) const {
        Raw r0 = raw(first, lane), r1 = raw(first + step, lane);
        for (int64_t b = first; b < blocks; b += step) {
            const Raw r2 = raw(b + 2 * step, lane);
            double w[EACH];
            weigh(r0, b, lane, w);
            f(b, wave_sum(sum(w)));
            r0 = r1;
            r1 = r2;
        }
    }
};

// the sum of n numbers over the workgroup's waves, each a run of them (part: its sum), in the same order every time
__device__ __forceinline__ double group_sum(const double *x, int64_t n, int wave, int lane, double *part) {
    const int64_t per = (n + WAVES - 1) / WAVES;
    double s = 0.0;
    for (int64_t b = wave * per + lane; b < (wave + 1) * per && b < n; b += 64) s += x[b];
    s = wave_sum(s);
    if (lane == 0) part[wave] = s;
    __syncthreads();
    s = 0.0;
    for (int k = 0; k < WAVES; ++k) s += part[k];
    return s;
}

template <typename E>
__device__ __forceinline__ Sampled<E> sampled_row(const VerifyParams &p, int64_t n, int i, int n_drafts, float top, double c) {
    const bool refused = i < n_drafts;
    int64_t d = -1;
    if (refused && !p.probs) d = p.drafts[n * p.K + i];
    return Sampled<E>{Row<E>(reinterpret_cast<const E *>(p.logits) + n * p.ld_stream + i * p.ld_row, p.V), p.V, top, c,
                      d >= 0 && d < p.V ? (int)d : -1, nullptr, p.probs_dtype, 0.0};
}
__device__ __forceinline__ int drafts_of(const VerifyParams &p, int64_t n) {
    const int k = p.n_drafts ? p.n_drafts[n] : p.K;
    return k < 0 ? 0 : k > p.K ? p.K : k;
}
__device__ __forceinline__ const void *probs_row(const VerifyParams &p, int64_t n, int i) {
    return reinterpret_cast<const char *>(p.probs) + (n * p.ld_probs_stream + i * p.ld_probs_row) * (p.probs_dtype == 0 ? 4 : 2);
}

}  // namespace

// Per stream, over gridDim.x workgroups: all decide how many drafts stand, and sum their blocks of the row that
// is sampled.  Three loads that wait for each other, two barriers, then some 30 instructions a logit, half of them
// in 64 bits: 8 us at 64 streams of 32,000 ids, 27-30 at 128 of 131,072.
template <typename E>
__global__ void __launch_bounds__(64 * WAVES) stand_kernel(const VerifyParams p) {
    __shared__ double zs[65], part[WAVES];
    __shared__ float tops[65];
    __shared__ int ats[65], verdict[65];
    const int tid = threadIdx.x, lane = tid & 63, K = p.K, V = p.V;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t n = blockIdx.y + (int64_t)blockIdx.z * gridDim.y, chunks = p.chunks, blocks = p.blocks;
    if (n >= p.N) return;
    const float t = p.temperature[n];
    const bool sampled = t > 0.f;
    if (!sampled && blockIdx.x > 0) return;
    const double c = sampled ? LOG2E / (double)t : 0.0;
    const int n_drafts = drafts_of(p, n);
    // what the decision takes of a draft, loaded beside the rows' chunks
    int64_t d = -1;
    float ud = 0.f, xd = 0.f;
    double qd = 1.0;
    if (tid < n_drafts) {
        d = p.drafts[n * K + tid];
        ud = p.uniforms[n * (K + 1) + tid];
        if (d >= 0 && d < V) {
            xd = (float)(reinterpret_cast<const E *>(p.logits) + n * p.ld_stream + tid * p.ld_row)[d];
            if (p.probs) qd = (double)param_f(probs_row(p, n, tid), p.probs_dtype, d);
        }
    }
    for (int i = wave; i <= n_drafts; i += WAVES) {                // every row's top and mass, a wave per row
        const RowMass *rows = p.rows + (n * (K + 1) + i) * chunks;
        float top = -__builtin_inff();
        int at = 0x7fffffff;
        double z = 0.0;
        if (chunks <= 64) {
            const RowMass r = lane < chunks ? rows[lane] : RowMass{0.f, top, -1};
            top = wave_max(r.at >= 0 ? r.top : top);
            if (r.at >= 0 && r.top == top) at = r.at;
            if (sampled && r.at >= 0) z = (double)r.sum * mass(r.top, top, c);
        } else {
            for (int64_t k = lane; k < chunks; k += 64)
                if (rows[k].at >= 0) top = fmaxf(top, rows[k].top);
            top = wave_max(top);
            for (int64_t k = lane; k < chunks; k += 64) {
                const RowMass r = rows[k];
                if (r.at >= 0 && r.top == top && r.at < at) at = r.at;
                if (sampled && r.at >= 0) z += (double)r.sum * mass(r.top, top, c);
            }
        }
        at = wave_min(at);
        z = wave_sum(z);
        if (lane == 0) {
            tops[i] = top;
            ats[i] = at;
            zs[i] = z;
        }
    }
    __syncthreads();
    // 1: the draft stands, 0: it does not, 2: too near to tell from an fp32 sum
    if (tid < n_drafts) {
        int v = 0;
        if (d >= 0 && d < V) {
            if (sampled) {
                const double w = mass(xd, tops[tid], c), lhs = (double)ud * qd * zs[tid];
                v = fabs(lhs - w) <= 1e-5 * w && w > 0.0 ? 2 : lhs < w ? 1 : 0;
            } else {
                v = d == ats[tid] && (double)ud * qd < 1.0 ? 1 : 0;
            }
        }
        verdict[tid] = v;
    }
    __syncthreads();
    int i = 0;
    double *sums = p.sums + n * 2 * blocks;
    for (;;) {
        while (i < n_drafts && verdict[i] == 1) ++i;
        const bool near = i < n_drafts && verdict[i] == 2;
        if (!near && !sampled) break;
        Sampled<E> row = sampled_row<E>(p, n, i, n_drafts, tops[i], c);
        if (near) row.without = -1;
        // the whole row in every workgroup where a draft is near, else this one's blocks: one copy of the code
        const int64_t first = near ? wave : (int64_t)blockIdx.x * WAVES + wave, step = near ? WAVES : (int64_t)gridDim.x * WAVES;
        double z = 0.0;
        row.sums(first, step, blocks, lane, [&](int64_t b, double s) __attribute__((always_inline)) {
            z += s;
            if (!near && lane == 0) sums[b] = s;
        });
        if (!near) break;
        if (lane == 0) part[wave] = z;
        __syncthreads();
        z = 0.0;
        for (int k = 0; k < WAVES; ++k) z += part[k];
        if (tid == i) verdict[i] = (double)ud * qd * z < mass(xd, tops[i], c) ? 1 : 0;
        __syncthreads();
    }
    if (blockIdx.x > 0) return;
    if (tid == 0) {
        p.stood[n] = Stood{i, tops[i]};
        p.accepted[n] = i;
    }
    for (int j = tid; j <= K; j += blockDim.x)                     // a sampled stream's token comes last
        p.tokens[n * (K + 1) + j] = j < i ? p.drafts[n * K + j] : j == i ? ats[i] : -1;
}

// What the draft's probabilities leave of a refused draft's row, in blocks.
template <typename E>
__global__ void __launch_bounds__(64 * WAVES) rest_kernel(const VerifyParams p) {
    __shared__ double part[WAVES];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t n = blockIdx.y + (int64_t)blockIdx.z * gridDim.y, blocks = p.blocks;
    if (n >= p.N) return;
    const float t = p.temperature[n];
    const Stood st = p.stood[n];
    const int n_drafts = drafts_of(p, n);
    if (!(t > 0.f) || st.count >= n_drafts) return;
    double *sums = p.sums + n * 2 * blocks;
    Sampled<E> row = sampled_row<E>(p, n, st.count, n_drafts, st.top, LOG2E / (double)t);
    row.q = probs_row(p, n, st.count);
    row.z = group_sum(sums, blocks, wave, lane, part);
    row.sums((int64_t)blockIdx.x * WAVES + wave, (int64_t)gridDim.x * WAVES, blocks, lane,
             [&](int64_t b, double s) __attribute__((always_inline)) {
                 if (lane == 0) sums[blocks + b] = s;
             });
}

// The token of a sampled stream: the first id at which the running sum passes u times the whole.
template <typename E>
__global__ void __launch_bounds__(64 * WAVES) choose_kernel(const VerifyParams p) {
    __shared__ double part[WAVES], part2[WAVES];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), K = p.K;
    const int64_t n = blockIdx.y + (int64_t)blockIdx.z * gridDim.y, blocks = p.blocks;
    if (n >= p.N) return;
    const float t = p.temperature[n];
    const Stood st = p.stood[n];
    const int n_drafts = drafts_of(p, n);
    const double u = (double)p.uniforms[n * (K + 1) + K];
    if (!(t > 0.f)) return;
    const double *sums = p.sums + n * 2 * blocks, *runs = part;
    Sampled<E> row = sampled_row<E>(p, n, st.count, n_drafts, st.top, LOG2E / (double)t);
    double whole = group_sum(sums, blocks, wave, lane, part);
    if (p.probs && st.count < n_drafts) {
        const double rest = group_sum(sums + blocks, blocks, wave, lane, part2);
        if (rest > 0.0) {                                          // else the draft's probabilities cover the row's
            row.q = probs_row(p, n, st.count);
            row.z = whole;
            whole = rest;
            sums += blocks;
            runs = part2;
        }
    }
    // the wave in whose run of blocks the sum passes; where rounding lets none, the last with any
    const double goal = u * whole;
    double before = 0.0, base = 0.0;
    int mine = -1;
    for (int k = 0; k < WAVES; ++k) {
        if (runs[k] > 0.0) {
            mine = k;
            base = before;
        }
        before += runs[k];
        if (runs[k] > 0.0 && before > goal) break;
    }
    if (wave != mine) return;
    const int64_t per = (blocks + WAVES - 1) / WAVES, end = (wave + 1) * per < blocks ? (wave + 1) * per : blocks;
    int64_t block = -1;
    double start = 0.0;
    bool passed = false;
    for (int64_t b0 = wave * per; b0 < end && !passed; b0 += 64) {
        const double own = b0 + lane < end ? sums[b0 + lane] : 0.0, upto = base + wave_prefix(own);
        const int l = passing_lane(own, upto, goal, passed);
        if (l >= 0) {
            block = b0 + l;
            start = lane_d(upto - own, l);
        }
        base = lane_d(upto, 63);
    }
    if (block < 0) return;
    double w[EACH];
    row.weigh(row.raw(block, lane), block, lane, w);
    const double own = row.sum(w), upto = start + wave_prefix(own);
    const int l = passing_lane(own, upto, goal, passed);
    double run = upto - own;
    int last = -1;
    bool over = false;
    unroll<EACH>([&](auto e) {
        run += w[e];
        if (w[e] > 0.0 && !over) {
            last = (int)(block * BLOCK + EACH * lane + e - row.row.first);
            over = run > goal;
        }
    });
    if (lane == l && last >= 0) p.tokens[n * (K + 1) + st.count] = last;
}

static int64_t verify_chunks(int64_t V) { return (V + 7 + CHUNK - 1) / CHUNK; }
static int64_t verify_blocks(int64_t V) { return (V + 7 + BLOCK - 1) / BLOCK; }

// the sampled rows' block sums (and what the draft leaves of them), the rows' chunks, the drafts that stand
int64_t verify_workspace(int64_t N, int64_t K, int64_t V) {
    return N * 2 * verify_blocks(V) * (int64_t)sizeof(double) + N * (K + 1) * verify_chunks(V) * (int64_t)sizeof(RowMass) +
           N * (int64_t)sizeof(Stood);
}

template <typename E> static void verify_typed(const VerifyParams &p, hipStream_t stream) {
    // rows and streams over two grid dimensions of at most 65,535: one dimension holds under 2^32 threads, 2^23 streams
    const int64_t rows = p.N * (p.K + 1), ry = rows < 32768 ? rows : 32768, ny = p.N < 32768 ? p.N : 32768;
    row_mass_kernel<E><<<dim3((unsigned)((p.chunks + ROW_WAVES - 1) / ROW_WAVES), (unsigned)ry, (unsigned)((rows + ry - 1) / ry)),
                         dim3(64 * ROW_WAVES), 0, stream>>>(p);
    // a block to a wave, up to SHARE workgroups of a decision's latency each (64 streams of 32,000: 8 each; 128 of 131,072: 4)
    const int64_t most = (p.blocks + WAVES - 1) / WAVES, share = SHARE / p.N > 1 ? SHARE / p.N : 1;
    const dim3 grid((unsigned)(most < share ? most : share), (unsigned)ny, (unsigned)((p.N + ny - 1) / ny));
    stand_kernel<E><<<grid, dim3(64 * WAVES), 0, stream>>>(p);
    if (p.probs) rest_kernel<E><<<grid, dim3(64 * WAVES), 0, stream>>>(p);
    choose_kernel<E><<<dim3(1, grid.y, grid.z), dim3(64 * WAVES), 0, stream>>>(p);
}

hipError_t verify_drafts(int dtype, VerifyParams p, void *workspace, hipStream_t stream) {
    p.chunks = verify_chunks(p.V);
    p.blocks = verify_blocks(p.V);
    p.sums = reinterpret_cast<double *>(workspace);
    p.rows = reinterpret_cast<RowMass *>(p.sums + p.N * 2 * p.blocks);
    p.stood = reinterpret_cast<Stood *>(p.rows + p.N * (p.K + 1) * p.chunks);
    if (dtype == 0) verify_typed<float>(p, stream);
    else if (dtype == 1) verify_typed<__bf16>(p, stream);
    else verify_typed<_Float16>(p, stream);
    return hipGetLastError();
}

namespace {

constexpr int LOOK_THREADS = 256, LOOK_EACH = 8;                   // places a thread has in flight
constexpr int64_t LOOK_RUN = 8192;                                 // places of a workgroup, at the least

__device__ __forceinline__ long long wave_best(long long x) {
    for (int m = 32; m; m >>= 1) {
        const long long y = __shfl_xor(x, m);
        x = y > x ? y : x;
    }
    return x;
}

// the drafts behind place best % 2^40 (best < 0: none), over the threads of a wave
template <typename I>
__device__ __forceinline__ void lookup_finish(const LookupParams &p, int64_t b, const I *text, int64_t n, long long best, int lane) {
    const int64_t start = (best & ((1LL << 40) - 1)) + 1;
    if (lane < p.K) p.drafts[b * p.K + lane] = best < 0 ? 0 : (int64_t)text[start + lane % (n - start)];
    if (lane == 0) p.counts[b] = best < 0 ? 0 : p.K;
}
__device__ __forceinline__ int64_t lookup_length(const LookupParams &p, int64_t b) {
    const int64_t n = p.lengths[b];
    return n < 0 ? 0 : n > p.cap ? p.cap : n;
}

}  // namespace

// Per stream: of all places e < n - 1 of its n tokens at which at least `shortest` of the last
// tokens end as well, the one where most of them do (up to `longest`), of those the last, as the
// largest 2^40 matches + e; the drafts are what follows it, again from there where the text ends.
// gridDim.x workgroups read a run of it each; a lone one finishes, else their bests are left
// for lookup_finish_kernel.  Bound by the text's read; a thread has eight places in flight (one after the
// other, 64 texts of 131,072: 215 us).
template <typename I>
__global__ void __launch_bounds__(LOOK_THREADS) lookup_kernel(const LookupParams p) {
    __shared__ long long keys[LOOK_THREADS / 64];
    const int tid = threadIdx.x, lane = tid & 63;
    const int64_t b = blockIdx.y + (int64_t)blockIdx.z * gridDim.y;
    if (b >= p.N) return;
    const I *text = reinterpret_cast<const I *>(p.history) + b * p.ld;
    const int64_t n = lookup_length(p, b);
    const int64_t first = blockIdx.x * p.run, end = first + p.run < n - 1 ? first + p.run : n - 1;
    long long best = -1;
    const I last = n > 0 ? text[n - 1] : (I)0;
    for (int64_t e0 = first; e0 < end; e0 += LOOK_THREADS * LOOK_EACH) {
        I here[LOOK_EACH];
        unroll<LOOK_EACH>([&](auto j) {
            const int64_t e = e0 + j * LOOK_THREADS + tid;
            here[j] = text[e < end ? e : end - 1];
        });
        unroll<LOOK_EACH>([&](auto j) {
            const int64_t e = e0 + j * LOOK_THREADS + tid;
            if (here[j] == last && e < end) {
                int m = 1;
                while (m < p.longest && m <= e && text[e - m] == text[n - 1 - m]) ++m;
                const long long key = ((long long)m << 40) | e;
                if (m >= p.shortest && key > best) best = key;
            }
        });
    }
    best = wave_best(best);
    if (lane == 0) keys[tid >> 6] = best;
    __syncthreads();
    if (tid >= 64) return;
    for (int k = 0; k < LOOK_THREADS / 64; ++k) best = keys[k] > best ? keys[k] : best;
    if (gridDim.x == 1) lookup_finish<I>(p, b, text, n, best, lane);
    else if (lane == 0) p.best[b * gridDim.x + blockIdx.x] = best;
}

template <typename I>
__global__ void __launch_bounds__(64) lookup_finish_kernel(const LookupParams p) {
    const int lane = threadIdx.x;
    const int64_t b = blockIdx.x;
    long long best = -1;
    for (int64_t k = lane; k < p.runs; k += 64) {
        const long long key = p.best[b * p.runs + k];
        best = key > best ? key : best;
    }
    best = wave_best(best);
    lookup_finish<I>(p, b, reinterpret_cast<const I *>(p.history) + b * p.ld, lookup_length(p, b), best, lane);
}

// Runs a text is read in: one of up to LOOK_RUN places (a second launch costs what they do), and above as many of that
// size as make 1,024 workgroups.
static int64_t lookup_runs(int64_t N, int64_t cap) {
    const int64_t most = (cap + LOOK_RUN - 1) / LOOK_RUN, share = 1024 / (N > 0 ? N : 1);
    const int64_t runs = most < share ? most : share;
    return runs > 1 ? runs : 1;
}
int64_t lookup_workspace(int64_t N, int64_t cap) {
    const int64_t runs = lookup_runs(N, cap);
    return runs > 1 ? N * runs * (int64_t)sizeof(long long) : 0;
}

template <typename I> static void lookup_typed(const LookupParams &p, hipStream_t stream) {
    const int64_t ny = p.N < 32768 ? p.N : 32768;
    lookup_kernel<I><<<dim3((unsigned)p.runs, (unsigned)ny, (unsigned)((p.N + ny - 1) / ny)), dim3(LOOK_THREADS), 0, stream>>>(p);
    if (p.runs > 1) lookup_finish_kernel<I><<<dim3((unsigned)p.N), dim3(64), 0, stream>>>(p);
}

hipError_t lookup_drafts(bool wide, LookupParams p, void *workspace, hipStream_t stream) {
    p.runs = lookup_runs(p.N, p.cap);
    p.run = (p.cap + p.runs - 1) / p.runs;
    p.best = reinterpret_cast<long long *>(workspace);
    if (wide) lookup_typed<int64_t>(p, stream);
    else lookup_typed<int32_t>(p, stream);
    return hipGetLastError();
}

}  // namespace vgdr
