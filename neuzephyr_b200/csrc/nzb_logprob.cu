// Log probabilities of given tokens with entropy and the top alternatives, and their gradient. Beside the softmax
// and binary-cross-entropy head: the loss of a model whose answer is one of `vocab` tokens.
//
// With z = scale x over a row: lse = ln sum exp z, logprob = z_t - lse, H = lse - sum p z. Everything is in powers of
// two, k = scale log2(e). One walk over the row: every thread keeps its largest logit m, s = sum e and w = sum e u with
// u = (x - m) k and e = 2^u; when m grows by d / k, u falls by d: w = f (w - d s), s = f s with f = 2^-d. Two such
// triples join the same way, so ln s and H = ln s - (w / s) ln 2 need no second walk and cancel nothing (w <= 0).
// Logits are read as no less than -2^27, so that a masked one (-inf, -1e9, the type's lowest) has e = 0 and e u = 0.
#include <cooperative_groups.h>

#include "nzb_elem.cuh"
#include "nzb_internal.h"

namespace nzb {

namespace cg = cooperative_groups;

constexpr float kEmpty = -134217728.f;  // -2^27, exact in bf16: a row without a logit above it has nothing left to choose from
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

// A 16-byte block of logits: -inf beyond the row.
template <typename T>
__device__ __forceinline__ uint4 load_logits(const T* row, int first, int n) {
    constexpr int VEC = Elem<T>::VEC;
    if (first >= 0 && first + VEC <= n) return __ldcs(reinterpret_cast<const uint4*>(row + first));
    union { uint4 u; T e[VEC]; } b;
#pragma unroll
    for (int i = 0; i < VEC; i++) b.e[i] = first + i >= 0 && first + i < n ? row[first + i] : Elem<T>::from(-INFINITY);
    return b.u;
}
// Largest element of a block, NaN left out (-inf if there is nothing else).
__device__ __forceinline__ float block_max(const uint4& u, float) {
    const float m = fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)), fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
    return m == m ? m : -INFINITY;
}
__device__ __forceinline__ float block_max(const uint4& u, __half) {
    const __half2* h = reinterpret_cast<const __half2*>(&u);
    const __half2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    const float f = fmaxf(__low2float(m), __high2float(m));
    return f == f ? f : -INFINITY;
}
__device__ __forceinline__ float block_max(const uint4& u, __nv_bfloat16) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
    const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    const float f = fmaxf(__low2float(m), __high2float(m));
    return f == f ? f : -INFINITY;
}
// The elements of a block as floats no less than kEmpty, NaN kept. bf16 has the range, so two are raised at once.
__device__ __forceinline__ void unpack_raised(const uint4& u, float (&f)[4], float) {
    Elem<float>::unpack(u, f);
#pragma unroll
    for (int i = 0; i < 4; i++) f[i] = max_nan(f[i], kEmpty);
}
__device__ __forceinline__ void unpack_raised(const uint4& u, float (&f)[8], __half) {
    Elem<__half>::unpack(u, f);
#pragma unroll
    for (int i = 0; i < 8; i++) f[i] = max_nan(f[i], kEmpty);
}
__device__ __forceinline__ void unpack_raised(const uint4& u, float (&f)[8], __nv_bfloat16) {
    uint4 r = u;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&r);
    const __nv_bfloat162 low = __float2bfloat162_rn(kEmpty);
#pragma unroll
    for (int i = 0; i < 4; i++) h[i] = __hmax2_nan(h[i], low);
    Elem<__nv_bfloat16>::unpack(r, f);
}

// Running sums of a part of a row.
struct RowSums {
    float top;   // largest logit, raised
    float s, w;  // sum e, sum e u
};
__device__ __forceinline__ RowSums join(const RowSums& a, const RowSums& b, float k) {
    RowSums j;
    j.top = fmaxf(a.top, b.top);
    const float ua = (a.top - j.top) * k, ub = (b.top - j.top) * k, fa = exp2_fast(ua), fb = exp2_fast(ub);
    j.s = fa * a.s + fb * b.s;
    j.w = fa * fmaf(ua, a.s, a.w) + fb * fmaf(ub, b.s, b.w);
    return j;
}

constexpr int kLogprobThreads = 256;  // per CTA; 64 for short rows
constexpr int kLogprobFly = 4;    // blocks in flight per thread
constexpr int kLogprobCluster = 8;  // CTAs that share a row, at most; lanes of a join too
constexpr int kTopMax = 32;
constexpr int kTopBuffer = 1024;  // candidates for the alternatives held in shared memory

// Order of the alternatives: larger logit first, then the lower column. NaN ranks last.
__device__ __forceinline__ bool ranks_before(float av, int ai, float bv, int bi) { return av > bv || (av == bv && ai < bi); }

template <typename T>
__device__ __forceinline__ float rank_value(T x) {
    const float f = Elem<T>::to(x);
    return f == f ? f : -INFINITY;
}

template <int NT>
struct TopSmem {
    float lane_max[NT];
    float value[kTopBuffer];
    int column[kTopBuffer];
    int chosen[NT];
    int count, n_chosen, overflow;
    float bound;
    float best_v[NT / 32];
    int best_i[NT / 32];
};

// Orders the first `count` candidates (at most kTopBuffer) and leaves the top_k best in front.
template <int NT>
__device__ __forceinline__ void rank_candidates(TopSmem<NT>& s, int count, int top_k) {
    constexpr int PER = kTopBuffer / NT;
    const int t = threadIdx.x;
    float v[PER];
    int col[PER], at[PER];
#pragma unroll
    for (int j = 0; j < PER; j++) {
        const int i = t + j * NT;
        at[j] = kTopBuffer;
        if (i >= count) continue;
        v[j] = s.value[i];
        col[j] = s.column[i];
        int before = 0;
        for (int o = 0; o < count; o++) before += ranks_before(s.value[o], s.column[o], v[j], col[j]);
        at[j] = before;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PER; j++) {
        if (at[j] < top_k) {
            s.value[at[j]] = v[j];
            s.column[at[j]] = col[j];
        }
    }
    __syncthreads();
}

// The part of a row that a CTA looks at. Whole 16-byte blocks [w0, w1) go round the threads: thread t has w0 + t,
// w0 + t + threads, ...; a first block that starts before the row is thread 0's too, a last one that ends behind it thread
// 1's (-1: there is none).
struct Stretch {
    int w0, w1, head, tail;
    int lead;
};
__device__ __forceinline__ Stretch make_stretch(int vocab, int lead, int vec, int part, int parts) {
    Stretch st;
    st.lead = lead;
    const int blocks = (vocab + lead + vec - 1) / vec, per = (blocks + parts - 1) / parts;
    const int b0 = min(blocks, part * per), b1 = min(blocks, b0 + per);
    const int first = lead ? 1 : 0, last = (vocab + lead) / vec;  // the row's whole blocks
    st.w0 = max(b0, first);
    st.w1 = max(st.w0, min(b1, last));
    st.head = b0 == 0 && b1 > 0 && (lead || last == 0) ? 0 : -1;
    st.tail = b1 == blocks && b1 > b0 && last < blocks && last > 0 ? last : -1;
    return st;
}

// The top_k-th largest of a CTA's NT values, by one warp: rounds of the largest one left.
template <int NT>
__device__ __forceinline__ float kth_largest(const float* value, int top_k, int lane) {
    uint32_t key[NT / 32], mine = 0;
#pragma unroll
    for (int j = 0; j < NT / 32; j++) {
        const uint32_t u = __float_as_uint(value[lane + 32 * j]);
        key[j] = u & 0x80000000u ? ~u : u | 0x80000000u;  // unsigned numbers in the floats' order
        mine = max(mine, key[j]);
    }
    uint32_t best = 0;
    for (int i = 0; i < top_k; i++) {
        best = __reduce_max_sync(0xffffffffu, mine);
        const uint32_t holders = __ballot_sync(0xffffffffu, mine == best);
        if (lane == __ffs(holders) - 1) {
            bool taken = false;
            mine = 0;
#pragma unroll
            for (int j = 0; j < NT / 32; j++) {
                if (!taken && key[j] == best) {
                    key[j] = 0;
                    taken = true;
                }
                mine = max(mine, key[j]);
            }
        }
    }
    return __uint_as_float(best & 0x80000000u ? best & 0x7fffffffu : ~best);
}

// The top_k largest logits of a stretch into s.value / s.column [0, top_k), in order; fewer than top_k elements are
// filled up with -inf in columns behind the row. lane_max[t] holds the largest of thread t's logits: the top_k-th
// largest of these is a lower bound of the top_k-th largest logit, so only the blocks of threads whose maximum
// reaches the bound are looked at again.
template <typename T, int NT>
__device__ void top_of_row(TopSmem<NT>& s, const T* row, int n, const Stretch& st, int top_k) {
    constexpr int VEC = Elem<T>::VEC;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int lead = st.lead;
    if (t == 0) s.count = s.n_chosen = 0;
    __syncthreads();
    const float mine = s.lane_max[t];
    if (warp == 0) {
        const float bound = kth_largest<NT>(s.lane_max, top_k, lane);
        if (lane == 0) s.bound = bound;
    }
    __syncthreads();
    const float bound = s.bound;
    if (mine >= bound) s.chosen[atomicAdd(&s.n_chosen, 1)] = t;
    __syncthreads();
    const auto look = [&](const uint4& u, int first) {
        if (!(block_max(u, T()) >= bound)) return;  // most blocks of a chosen thread hold nothing of interest
        union { uint4 u; T e[VEC]; } x;
        x.u = u;
#pragma unroll
        for (int i = 0; i < VEC; i++) {
            const int col = first + i;
            const float v = rank_value(x.e[i]);
            if (v >= bound && col >= 0 && col < n) {
                const int at = atomicAdd(&s.count, 1);
                if (at < kTopBuffer) {
                    s.value[at] = v;
                    s.column[at] = col;
                }
            }
        }
    };
    for (int c = warp; c < s.n_chosen; c += NT / 32) {
        const int who = s.chosen[c];
        for (int b = st.w0 + who + lane * NT; b < st.w1; b += 32 * NT) look(*reinterpret_cast<const uint4*>(row + (b * VEC - lead)), b * VEC - lead);
        const int cut = who == 0 ? st.head : who == 1 ? st.tail : -1;
        if (lane == 0 && cut >= 0) look(load_logits(row, cut * VEC - lead, n), cut * VEC - lead);
    }
    __syncthreads();
    const int c0 = st.head >= 0 ? 0 : st.w0 * VEC - lead, c1 = st.tail >= 0 || st.w1 <= st.w0 ? n : st.w1 * VEC - lead;
    int count = s.count;
    if (count <= kTopBuffer) {
        __syncthreads();
        if (count < top_k) {
            if (t < top_k - count) {
                s.value[count + t] = -INFINITY;
                s.column[count + t] = n + count + t;
            }
            count = top_k;
            __syncthreads();
        }
        rank_candidates(s, count, top_k);
        return;
    }
    // Too many logits reach the bound (long runs of equal ones): take the alternatives one after the other, each the
    // best of those that rank behind the one before.
    float last_v = INFINITY;
    int last_i = -1;
    for (int k = 0; k < top_k; k++) {
        float bv = -INFINITY;
        int bi = n;
        for (int c = c0 + t; c < c1; c += NT) {
            const float v = rank_value(row[c]);
            if (ranks_before(last_v, last_i, v, c) && ranks_before(v, c, bv, bi)) {
                bv = v;
                bi = c;
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const float ov = __shfl_xor_sync(0xffffffffu, bv, o);
            const int oi = __shfl_xor_sync(0xffffffffu, bi, o);
            if (ranks_before(ov, oi, bv, bi)) {
                bv = ov;
                bi = oi;
            }
        }
        if (lane == 0) {
            s.best_v[warp] = bv;
            s.best_i[warp] = bi;
        }
        __syncthreads();
        bv = s.best_v[0];
        bi = s.best_i[0];
        for (int w = 1; w < NT / 32; w++)
            if (ranks_before(s.best_v[w], s.best_i[w], bv, bi)) {
                bv = s.best_v[w];
                bi = s.best_i[w];
            }
        if (t == 0) {
            s.value[k] = bv;
            s.column[k] = bi;
        }
        last_v = bv;
        last_i = bi;
        __syncthreads();
    }
}

// A row per CTA, or per cluster of CTAs when there are few rows: each takes a stretch of the row, and the first one
// joins what the others left in their shared memory.
template <typename T, typename Index, int NT, bool CLUSTER>
__global__ void __launch_bounds__(NT)
token_logprob_kernel(const T* __restrict__ logits, const Index* __restrict__ targets, float* __restrict__ logprob,
                     float* __restrict__ entropy, float* __restrict__ lse_out, float* __restrict__ top_logprob,
                     Index* __restrict__ top_index, int vocab, int64_t ld, float scale, int top_k, int parts) {
    constexpr int VEC = Elem<T>::VEC, FLY = kLogprobFly, WARPS = NT / 32;
    __shared__ RowSums warp_sums[WARPS];
    __shared__ RowSums cta_sums;
    __shared__ TopSmem<NT> top;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int part = CLUSTER ? blockIdx.x % parts : 0;
    const int64_t r = CLUSTER ? blockIdx.x / parts : blockIdx.x;
    const T* row = logits + r * ld;
    const int lead = row_lead(row);
    const Stretch st = make_stretch(vocab, lead, VEC, part, CLUSTER ? parts : 1);
    const float k = scale * kLog2e;
    const float2 k2 = make_float2(k, k);
    RowSums a = {kEmpty, 0.f, 0.f};
    float seen = -INFINITY;  // largest logit of this thread's, NaN left out
    float2 s2 = make_float2(0.f, 0.f), w2 = s2;
    const auto take = [&](const auto& u) {
        constexpr int N = sizeof(u) / sizeof(uint4);
        float mx = block_max(u[0], T());
#pragma unroll
        for (int f = 1; f < N; f++) mx = fmaxf(mx, block_max(u[f], T()));
        seen = fmaxf(seen, mx);
        if (mx > a.top) {
            const float d = (a.top - mx) * k, fac = exp2_fast(d);
            w2 = make_float2(fac * fmaf(d, s2.x, w2.x), fac * fmaf(d, s2.y, w2.y));
            s2 = make_float2(fac * s2.x, fac * s2.y);
            a.top = mx;
        }
        const float2 minus = make_float2(-a.top, -a.top);
#pragma unroll
        for (int f = 0; f < N; f++) {
            float x[VEC];
            unpack_raised(u[f], x, T());
#pragma unroll
            for (int i = 0; i < VEC; i += 2) {
                const float2 v = mul2(add2(make_float2(x[i], x[i + 1]), minus), k2);
                const float2 e = make_float2(exp2_fast(v.x), exp2_fast(v.y));
                s2 = add2(s2, e);
                w2 = fma2(e, v, w2);
            }
        }
    };
    // whole blocks without any check, FLY of them in flight; the last round's missing ones as masked logits
    const uint4* at = reinterpret_cast<const uint4*>(row + st.w0 * VEC - lead) + t;
    int left = (st.w1 - st.w0 - t + NT - 1) / NT;  // of this thread
    for (; left >= FLY; left -= FLY, at += FLY * NT) {
        uint4 u[FLY];
#pragma unroll
        for (int f = 0; f < FLY; f++) u[f] = __ldcs(at + f * NT);
        take(u);
    }
    if (left > 0) {
        union { T e[VEC]; uint4 u; } none;
#pragma unroll
        for (int i = 0; i < VEC; i++) none.e[i] = Elem<T>::from(-INFINITY);
        uint4 u[FLY - 1];
#pragma unroll
        for (int f = 0; f < FLY - 1; f++) u[f] = f < left ? __ldcs(at + f * NT) : none.u;
        take(u);
    }
    const int cut = t == 0 ? st.head : t == 1 ? st.tail : -1;
    if (cut >= 0) {
        const uint4 u[1] = {load_logits(row, cut * VEC - lead, vocab)};
        take(u);
    }
    a.s = s2.x + s2.y;
    a.w = w2.x + w2.y;
    if (top_k) top.lane_max[t] = seen;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        RowSums b;
        b.top = __shfl_xor_sync(0xffffffffu, a.top, o);
        b.s = __shfl_xor_sync(0xffffffffu, a.s, o);
        b.w = __shfl_xor_sync(0xffffffffu, a.w, o);
        // both lanes of a pair join in the same order, so that they agree
        a = lane & o ? join(b, a, k) : join(a, b, k);
    }
    if (lane == 0) warp_sums[warp] = a;
    __syncthreads();
    // lanes 0..7 of the first warp hold the warps' (or, below, the CTAs') sums and join in pairs
    const auto join_eight = [&](RowSums a) {
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) {
            RowSums b;
            b.top = __shfl_down_sync(0xffu, a.top, o);
            b.s = __shfl_down_sync(0xffu, a.s, o);
            b.w = __shfl_down_sync(0xffu, a.w, o);
            a = join(a, b, k);
        }
        return a;
    };
    if (t < 8) {
        const RowSums none = {kEmpty, 0.f, 0.f};
        a = join_eight(t < WARPS ? warp_sums[t] : none);
        if (t == 0) cta_sums = a;
    }
    if (top_k) top_of_row(top, row, vocab, st, top_k);
    if (CLUSTER) {
        cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        if (part == 0) {
            if (t < 8) {
                const RowSums none = {kEmpty, 0.f, 0.f};
                a = join_eight(t < parts ? *cluster.map_shared_rank(&cta_sums, t) : none);
                __syncwarp(0xffu);
                if (t == 0) cta_sums = a;
            }
            if (top_k) {
                for (int i = top_k + t; i < top_k * parts; i += NT) {
                    const int p = i / top_k, j = i - p * top_k;
                    top.value[i] = *cluster.map_shared_rank(&top.value[j], p);
                    top.column[i] = *cluster.map_shared_rank(&top.column[j], p);
                }
                __syncthreads();
                rank_candidates(top, top_k * parts, top_k);
            }
        }
        cluster.sync();  // nobody leaves while the first CTA may still read
        if (part) return;
    }
    __syncthreads();
    const RowSums all = cta_sums;
    const bool empty = all.top <= kEmpty && all.s == all.s;
    const float ln_s = logf(all.s);  // not log2f times ln 2: two more roundings, the first in a coarser place
    if (t == 0) {
        if (lse_out) lse_out[r] = empty ? -INFINITY : fmaf(all.top, scale, ln_s);
        // a sum w of NaN beside a finite s: a logit so large (above 2^126) that u left fp32's range. Then every e is 0 or 1
        if (entropy) entropy[r] = empty ? 0.f : fmaf(all.w == all.w || all.s != all.s ? all.w / all.s : 0.f, -kLn2, ln_s);
        if (logprob) {
            const int64_t tgt = static_cast<int64_t>(targets[r]);
            float lp = 0.f;
            if (tgt >= 0 && tgt < vocab) lp = empty ? -INFINITY : fmaf(Elem<T>::to(row[tgt]) - all.top, scale, -ln_s);
            logprob[r] = lp;
        }
    }
    if (t < top_k) {
        if (top_logprob) top_logprob[r * top_k + t] = empty ? -INFINITY : fmaf(top.value[t] - all.top, scale, -ln_s);
        if (top_index) top_index[r * top_k + t] = static_cast<Index>(top.column[t]);
    }
}

// dlogits = scale (dl (1[target] - p) - dH p (ln p + H)), p = e^q with q = z - lse in one rounding (ln p near 0 counts).
template <typename T, typename Index, bool ENTROPY>
__global__ void __launch_bounds__(256)
token_logprob_backward_kernel(const T* logits, const Index* __restrict__ targets, const float* __restrict__ lse,
                              const float* __restrict__ entropy, const float* __restrict__ dlogprob,
                              const float* __restrict__ dentropy, T* dlogits, int vocab, int64_t ld, int64_t ld_d, float scale) {
    constexpr int VEC = Elem<T>::VEC, FLY = kLogprobFly;
    const int64_t r = blockIdx.y;
    const T* row = logits + r * ld;
    T* out = dlogits + r * ld_d;
    const int lead = row_lead(row);
    const int blocks = (vocab + lead + VEC - 1) / VEC;
    const int b0 = blockIdx.x * (256 * FLY) + threadIdx.x;
    uint4 u[FLY];
#pragma unroll
    for (int f = 0; f < FLY; f++)
        if (b0 + f * 256 < blocks) u[f] = load_logits(row, (b0 + f * 256) * VEC - lead, vocab);
    const bool same = row_lead(out) == lead;
    const int64_t tgt = static_cast<int64_t>(targets[r]);
    const bool has = tgt >= 0 && tgt < vocab;
    const float l = lse[r], dl = dlogprob && has ? dlogprob[r] : 0.f, dh = ENTROPY ? dentropy[r] : 0.f, H = ENTROPY ? entropy[r] : 0.f;
    const bool empty = l == -INFINITY;
    const float c0 = empty ? 0.f : -scale * (dl + dh * H), c1 = empty ? 0.f : -scale * dh;
    const float base = empty ? 0.f : -l;
    const float2 scale2 = make_float2(scale, scale), base2 = make_float2(base, base), log2e2 = make_float2(kLog2e, kLog2e), c02 = make_float2(c0, c0), c12 = make_float2(c1, c1);
#pragma unroll
    for (int f = 0; f < FLY; f++) {
        const int b = b0 + f * 256, first = b * VEC - lead;
        if (b >= blocks) break;
        float x[VEC];
        if (ENTROPY) unpack_raised(u[f], x, T());  // p ln p of a masked logit is 0
        else Elem<T>::unpack(u[f], x);
#pragma unroll
        for (int i = 0; i < VEC; i += 2) {
            const float2 q = fma2(make_float2(x[i], x[i + 1]), scale2, base2), q2 = mul2(q, log2e2);
            const float2 p = make_float2(exp2_fast(q2.x), exp2_fast(q2.y));
            const float2 d = mul2(p, ENTROPY ? fma2(c12, q, c02) : c02);
            x[i] = d.x;
            x[i + 1] = d.y;
        }
        if (empty) {
#pragma unroll
            for (int i = 0; i < VEC; i++) x[i] = 0.f;
        } else if (has && tgt >= first && tgt < first + VEC) {
#pragma unroll
            for (int i = 0; i < VEC; i++)
                if (first + i == tgt) x[i] = fmaf(scale, dl, x[i]);
        }
        if (same) {
            store_block(out, first, vocab, Elem<T>::pack(x));
        } else {
#pragma unroll
            for (int i = 0; i < VEC; i++)
                if (first + i >= 0 && first + i < vocab) out[first + i] = Elem<T>::from(x[i]);
        }
    }
}

template <typename T, typename Index>
static int launch_logprob(const nzb_token_logprob_desc* d, const void* logits, const void* targets, float* logprob, float* entropy,
                          float* lse, float* top_logprob, void* top_index, int top_k, int sm_count, cudaStream_t s) {
    const int64_t blocks = (d->vocab + Elem<T>::VEC - 1) / Elem<T>::VEC;
    // few rows: more CTAs share one, as long as each thread keeps a round of blocks; many short ones: smaller CTAs, whose
    // joins and selections are shorter (5000 x 3000 bf16 with four alternatives: 48 us by 256 threads)
    int parts = 1;
    while (parts < kLogprobCluster && d->rows * parts < 2 * sm_count && blocks >= (int64_t)parts * 2 * kLogprobThreads * kLogprobFly) parts *= 2;
    const bool small = parts == 1 && blocks < kLogprobThreads * kLogprobFly;
    if (d->rows * parts > INT32_MAX) return fail(NZB_ERR_UNSUPPORTED, "too many rows");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(d->rows * parts));
    cfg.blockDim = dim3(small ? 64 : kLogprobThreads);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = parts;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = parts > 1 ? 1 : 0;
    const auto kernel = parts > 1 ? token_logprob_kernel<T, Index, kLogprobThreads, true>
                        : small   ? token_logprob_kernel<T, Index, 64, false>
                                  : token_logprob_kernel<T, Index, kLogprobThreads, false>;
    NZB_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, static_cast<const T*>(logits), static_cast<const Index*>(targets), logprob, entropy,
                                    lse, top_logprob, static_cast<Index*>(top_index), (int)d->vocab, d->ld_logits, d->scale, top_k, parts));
    return NZB_OK;
}

static int check_logprob(const nzb_token_logprob_desc* d) {
    if (!d) return fail(NZB_ERR_BAD_ARG, "descriptor is null");
    if (d->rows < 0 || d->vocab < 0) return fail(NZB_ERR_BAD_ARG, "negative extent");
    if (d->rows > 65535ll * 32768 || d->vocab > (1 << 28)) return fail(NZB_ERR_UNSUPPORTED, "vocab at most 2^28, rows below 2^31");
    if (!known_dtype(d->dtype)) return fail(NZB_ERR_BAD_ARG, "unknown element type");
    if (d->index_type != NZB_I32 && d->index_type != NZB_I64) return fail(NZB_ERR_BAD_ARG, "unknown index type");
    // below 1e-4 a masked logit's 2^27 would leave it a probability
    if (!(d->scale >= 1e-4f) || d->scale > 1e6f) return fail(NZB_ERR_BAD_ARG, "scale must be in [1e-4, 1e6]");
    if (d->ld_logits < d->vocab) return fail(NZB_ERR_BAD_ARG, "leading dimension smaller than the row length");
    return NZB_OK;
}

}  // namespace nzb

using namespace nzb;

extern "C" {

int nzb_token_logprob_forward(const nzb_token_logprob_desc* d, const void* logits, const void* targets, float* logprob,
                              float* entropy, float* lse, float* top_logprob, void* top_index, void* stream) {
    int rc = check_logprob(d);
    if (rc != NZB_OK) return rc;
    if (d->top_k < 0 || d->top_k > kTopMax || d->top_k > d->vocab) return fail(NZB_ERR_BAD_ARG, "top_k must be in [0, 32] and at most vocab");
    if (d->rows == 0) return NZB_OK;
    if (d->vocab == 0) return fail(NZB_ERR_UNSUPPORTED, "vocab = 0 is not supported");
    if (!logits || (logprob && !targets)) return fail(NZB_ERR_BAD_ARG, "logits and targets must be non-null");
    if (!aligned_to(logits, dtype_size(d->dtype)) || !aligned_to(targets, index_size(d->index_type)) || !aligned_to(top_index, index_size(d->index_type))) return fail(NZB_ERR_BAD_ARG, "pointer is not a multiple of its element's size");
    DeviceState* ds;
    rc = get_device_state(&ds);
    if (rc != NZB_OK) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int top_k = top_logprob || top_index ? d->top_k : 0;
    NZB_DISPATCH_DTYPE(d->dtype, T, {
        rc = d->index_type == NZB_I64 ? launch_logprob<T, int64_t>(d, logits, targets, logprob, entropy, lse, top_logprob, top_index, top_k, ds->sm_count, s)
                                      : launch_logprob<T, int32_t>(d, logits, targets, logprob, entropy, lse, top_logprob, top_index, top_k, ds->sm_count, s);
    });
    return rc;
}

int nzb_token_logprob_backward(const nzb_token_logprob_desc* d, const void* logits, const void* targets, const float* lse,
                               const float* entropy, const float* dlogprob, const float* dentropy, void* dlogits, void* stream) {
    int rc = check_logprob(d);
    if (rc != NZB_OK) return rc;
    if (d->ld_dlogits < d->vocab) return fail(NZB_ERR_BAD_ARG, "leading dimension smaller than the row length");
    if (d->rows == 0 || d->vocab == 0) return NZB_OK;
    if (!logits || !targets || !lse || !dlogits || (dentropy && !entropy))
        return fail(NZB_ERR_BAD_ARG, "logits, targets, lse, dlogits (and entropy beside dentropy) must be non-null");
    if (logits == dlogits && d->ld_logits != d->ld_dlogits) return fail(NZB_ERR_BAD_ARG, "dlogits in place of logits needs their leading dimension");
    const int64_t size = dtype_size(d->dtype);
    if (!aligned_to(logits, size) || !aligned_to(dlogits, size) || !aligned_to(targets, index_size(d->index_type))) return fail(NZB_ERR_BAD_ARG, "pointer is not a multiple of its element's size");
    DeviceState* ds;
    rc = get_device_state(&ds);
    if (rc != NZB_OK) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    NZB_DISPATCH_DTYPE(d->dtype, T, {
        const int64_t blocks = (d->vocab + Elem<T>::VEC - 1) / Elem<T>::VEC + 1;
        const int64_t gx = (blocks + 256 * kLogprobFly - 1) / (256 * kLogprobFly);
        for (int64_t r0 = 0; r0 < d->rows; r0 += 65535) {
            const int64_t n = d->rows - r0 < 65535 ? d->rows - r0 : 65535;
            const dim3 grid((unsigned)gx, (unsigned)n);
            const T* x = static_cast<const T*>(logits) + r0 * d->ld_logits;
            T* o = static_cast<T*>(dlogits) + r0 * d->ld_dlogits;
            const float* ent = dentropy ? entropy + r0 : nullptr;
            const float* dlp = dlogprob ? dlogprob + r0 : nullptr;
            const float* dent = dentropy ? dentropy + r0 : nullptr;
            const auto launch = [&](auto kernel, auto index) {
                kernel<<<grid, 256, 0, s>>>(x, static_cast<const decltype(index)*>(targets) + r0, lse + r0, ent, dlp, dent, o, (int)d->vocab, d->ld_logits, d->ld_dlogits, d->scale);
            };
            if (d->index_type == NZB_I64) launch(dentropy ? token_logprob_backward_kernel<T, int64_t, true> : token_logprob_backward_kernel<T, int64_t, false>, int64_t());
            else launch(dentropy ? token_logprob_backward_kernel<T, int32_t, true> : token_logprob_backward_kernel<T, int32_t, false>, int32_t());
        }
    });
    NZB_CUDA_TRY(cudaGetLastError());
    return NZB_OK;
}

}  // extern "C"
