// Log probabilities of given tokens with entropy and the top alternatives, and their gradient. Beside the softmax
// and binary-cross-entropy head: the loss of a model whose answer is one of `vocab` tokens.
//
// With z = scale x over a row: lse = ln sum exp z, logprob = z_t - lse, H = lse - sum p z.
// One walk over the row: every thread keeps the running maximum m of its logits, s = sum e and w = sum e u with
// u = (x - m) scale and e = exp u; when m grows by d, w = f (w + d s) and s = f s with f = exp(d), d < 0. Two such
// triples join the same way, so ln s and H = ln s - w / s need no second walk and cancel nothing (w <= 0).
#include "nzb_internal.h"
#include "nzb_elem.cuh"

namespace nzb {

constexpr float kEmptyRow = -1e30f;  // a row without a z above this has nothing left to choose from
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kLowest = -3.402823466e38f;

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

// Running sums of a part of a row. u is in units of ln 2 / scale: u2 = (x - m) scale log2(e).
struct RowSums {
    float m, s, w;  // m: largest logit (unscaled); w = sum e * u2
};
__device__ __forceinline__ RowSums join(const RowSums& a, const RowSums& b, float k) {
    RowSums r;
    r.m = fmaxf(a.m, b.m);
    // differences of finite numbers, at worst -inf; clamped so that 0 * u stays 0
    const float ua = fmaxf((a.m - r.m) * k, -1000.f), ub = fmaxf((b.m - r.m) * k, -1000.f);
    const float fa = exp2_fast(ua), fb = exp2_fast(ub);
    r.s = a.s * fa + b.s * fb;
    r.w = fa * (a.w + ua * a.s) + fb * (b.w + ub * b.s);
    return r;
}

constexpr int kLogprobThreads = 256;
constexpr int kTopMax = 32;
constexpr int kTopBuffer = 1024;  // candidates for the alternatives held in shared memory

// Order of the alternatives: larger logit first, then the lower column. NaN ranks last.
__device__ __forceinline__ bool ranks_before(float av, int ai, float bv, int bi) { return av > bv || (av == bv && ai < bi); }

template <typename T>
__device__ __forceinline__ float rank_value(T x) {
    const float f = Elem<T>::to(x);
    return f == f ? f : -INFINITY;
}

struct TopSmem {
    float lane_max[kLogprobThreads];
    float value[kTopBuffer];
    int column[kTopBuffer];
    int chosen[kLogprobThreads];
    int count, n_chosen, overflow;
    float bound;
    float best_v[kLogprobThreads / 32];
    int best_i[kLogprobThreads / 32];
};

// The top_k largest logits of a row into s.value / s.column [0, top_k), in order. lane_max[t] holds the largest
// logit among the blocks t, t + threads, ... of the row: the top_k-th largest of these is a lower bound of the
// top_k-th largest logit, so only the blocks of threads whose maximum reaches the bound are looked at again.
template <typename T>
__device__ void top_of_row(TopSmem& s, const T* row, int n, int lead, int blocks, int top_k) {
    constexpr int VEC = Elem<T>::VEC, NT = kLogprobThreads;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    if (t == 0) {
        s.count = s.n_chosen = 0;
        s.bound = -INFINITY;
    }
    __syncthreads();
    const float mine = s.lane_max[t];
    int rank = 0;
    for (int i = 0; i < NT; i++) rank += ranks_before(s.lane_max[i], i, mine, t);
    if (rank == top_k - 1) s.bound = mine;
    __syncthreads();
    const float bound = s.bound;
    if (mine >= bound) s.chosen[atomicAdd(&s.n_chosen, 1)] = t;
    __syncthreads();
    for (int c = warp; c < s.n_chosen; c += NT / 32) {
        for (int b = s.chosen[c] + lane * NT; b < blocks; b += 32 * NT) {
            const int first = b * VEC - lead;
            union { uint4 u; T e[VEC]; } x;
            x.u = load_block(row, first, n);
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                const int col = first + i;
                const float v = rank_value(x.e[i]);
                if (col >= 0 && col < n && v >= bound) {
                    const int at = atomicAdd(&s.count, 1);
                    if (at < kTopBuffer) {
                        s.value[at] = v;
                        s.column[at] = col;
                    }
                }
            }
        }
    }
    __syncthreads();
    const int count = s.count;
    if (count <= kTopBuffer) {
        // at least top_k candidates: each finds its rank among them
        constexpr int PER = kTopBuffer / NT;
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
        return;
    }
    // Too many logits reach the bound (long runs of equal ones): take the alternatives one after the other, each the
    // best of those that rank behind the one before.
    float last_v = INFINITY;
    int last_i = -1;
    for (int k = 0; k < top_k; k++) {
        float bv = -INFINITY;
        int bi = n;
        for (int c = t; c < n; c += NT) {
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

template <typename T, typename Index>
__global__ void __launch_bounds__(kLogprobThreads)
token_logprob_kernel(const T* __restrict__ logits, const Index* __restrict__ targets, float* __restrict__ logprob,
                     float* __restrict__ entropy, float* __restrict__ lse_out, float* __restrict__ top_logprob,
                     Index* __restrict__ top_index, int vocab, int64_t ld, float scale, int top_k) {
    constexpr int VEC = Elem<T>::VEC, NT = kLogprobThreads;
    __shared__ RowSums warp_sums[NT / 32];
    __shared__ RowSums row_sums;
    __shared__ TopSmem top;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int64_t r = blockIdx.x;
    const T* row = logits + r * ld;
    const int lead = row_lead(row);
    const int blocks = (vocab + lead + VEC - 1) / VEC;
    const float k = scale * kLog2e;
    RowSums a = {kLowest, 0.f, 0.f};
    float seen = -INFINITY;  // largest logit of this thread's, NaN left out
    for (int b = t; b < blocks; b += NT) {
        const int first = b * VEC - lead;
        float f[VEC];
        if (first >= 0 && first + VEC <= vocab) {
            Elem<T>::unpack(*reinterpret_cast<const uint4*>(row + first), f);
        } else {
#pragma unroll
            for (int i = 0; i < VEC; i++) f[i] = first + i >= 0 && first + i < vocab ? Elem<T>::to(row[first + i]) : -INFINITY;
        }
        float mx = f[0];
#pragma unroll
        for (int i = 1; i < VEC; i++) mx = fmaxf(mx, f[i]);
        seen = fmaxf(seen, mx);
        if (mx > a.m) {
            const float u = fmaxf((a.m - mx) * k, -1000.f), fac = exp2_fast(u);
            a.w = fac * (a.w + u * a.s);
            a.s *= fac;
            a.m = mx;
        }
#pragma unroll
        for (int i = 0; i < VEC; i++) {
            const float u = max_nan((f[i] - a.m) * k, -1000.f);
            const float e = exp2_fast(u);
            a.s += e;
            a.w = fmaf(e, u, a.w);
        }
    }
    if (top_k) top.lane_max[t] = seen;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        RowSums b;
        b.m = __shfl_xor_sync(0xffffffffu, a.m, o);
        b.s = __shfl_xor_sync(0xffffffffu, a.s, o);
        b.w = __shfl_xor_sync(0xffffffffu, a.w, o);
        // both lanes of a pair join in the same order, so that they agree
        a = lane & o ? join(b, a, k) : join(a, b, k);
    }
    if (lane == 0) warp_sums[warp] = a;
    __syncthreads();
    if (t == 0) {
        for (int w = 1; w < NT / 32; w++) a = join(a, warp_sums[w], k);
        row_sums = a;
        const bool empty = a.m * scale <= kEmptyRow || a.s == 0.f;
        const float log_s = logf(a.s);
        if (lse_out) lse_out[r] = empty ? (a.s == a.s ? -INFINITY : a.s) : a.m * scale + log_s;
        if (entropy) entropy[r] = empty ? (a.s == a.s ? 0.f : a.s) : log_s - a.w / a.s * kLn2;
        if (logprob) {
            const int64_t tgt = static_cast<int64_t>(targets[r]);
            float lp = 0.f;
            if (tgt >= 0 && tgt < vocab) lp = empty ? (a.s == a.s ? -INFINITY : a.s) : (Elem<T>::to(row[tgt]) - a.m) * scale - log_s;
            logprob[r] = lp;
        }
    }
    if (!top_k) return;
    __syncthreads();
    top_of_row(top, row, vocab, lead, blocks, top_k);
    const RowSums all = row_sums;
    if (t < top_k) {
        const bool empty = all.m * scale <= kEmptyRow || all.s == 0.f;
        if (top_logprob) top_logprob[r * top_k + t] = empty && all.s == all.s ? -INFINITY : (top.value[t] - all.m) * scale - logf(all.s);
        if (top_index) top_index[r * top_k + t] = static_cast<Index>(top.column[t]);
    }
}

// dlogits = scale (dl (1[target] - p) - dH p (ln p + H)), p = exp(z - lse).
template <typename T, typename Index>
__global__ void __launch_bounds__(256)
token_logprob_backward_kernel(const T* logits, const Index* __restrict__ targets, const float* __restrict__ lse,
                              const float* __restrict__ entropy, const float* __restrict__ dlogprob,
                              const float* __restrict__ dentropy, T* dlogits, int vocab, int64_t ld, int64_t ld_d, float scale) {
    constexpr int VEC = Elem<T>::VEC;
    const int64_t r = blockIdx.y;
    const T* row = logits + r * ld;
    T* out = dlogits + r * ld_d;
    const int lead = row_lead(row);
    const bool same = row_lead(out) == lead;
    const int blocks = (vocab + lead + VEC - 1) / VEC;
    const int64_t tgt = static_cast<int64_t>(targets[r]);
    const bool has = tgt >= 0 && tgt < vocab;
    const float l = lse[r], dl = dlogprob && has ? dlogprob[r] : 0.f, dh = dentropy ? dentropy[r] : 0.f, H = dentropy ? entropy[r] : 0.f;
    const bool empty = l <= kEmptyRow;
    const float c0 = -scale * (dl + dh * H), c1 = -scale * dh;
    for (int b = blockIdx.x * 256 + threadIdx.x; b < blocks; b += gridDim.x * 256) {
        const int first = b * VEC - lead;
        float f[VEC];
        Elem<T>::unpack(load_block(row, first, vocab), f);
#pragma unroll
        for (int i = 0; i < VEC; i++) {
            const float q = max_nan(fmaf(f[i], scale, -l), -1000.f);  // ln p
            const float p = exp2_fast(q * kLog2e);
            f[i] = empty ? 0.f : p * fmaf(c1, q, c0);
            if (first + i == tgt && has && !empty) f[i] += scale * dl;
        }
        if (same) {
            store_block(out, first, vocab, Elem<T>::pack(f));
        } else {
#pragma unroll
            for (int i = 0; i < VEC; i++)
                if (first + i >= 0 && first + i < vocab) out[first + i] = Elem<T>::from(f[i]);
        }
    }
}

static int check_logprob(const nzb_token_logprob_desc* d) {
    if (!d) return fail(NZB_ERR_BAD_ARG, "descriptor is null");
    if (d->rows < 0 || d->vocab < 0) return fail(NZB_ERR_BAD_ARG, "negative extent");
    if (d->rows > 65535ll * 32768 || d->vocab > (1 << 28)) return fail(NZB_ERR_UNSUPPORTED, "vocab at most 2^28, rows below 2^31");
    if (!known_dtype(d->dtype)) return fail(NZB_ERR_BAD_ARG, "unknown element type");
    if (d->index_type != NZB_I32 && d->index_type != NZB_I64) return fail(NZB_ERR_BAD_ARG, "unknown index type");
    if (!(d->scale > 0.f) || d->scale > 1e6f) return fail(NZB_ERR_BAD_ARG, "scale must be in (0, 1e6]");
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
    if (!aligned_to(logits, dtype_size(d->dtype))) return fail(NZB_ERR_BAD_ARG, "pointer is not a multiple of its element's size");
    DeviceState* ds;
    rc = get_device_state(&ds);
    if (rc != NZB_OK) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int top_k = top_logprob || top_index ? d->top_k : 0;
    NZB_DISPATCH_DTYPE(d->dtype, T, {
        const T* x = static_cast<const T*>(logits);
        if (d->index_type == NZB_I64)
            token_logprob_kernel<T, int64_t><<<(unsigned)d->rows, kLogprobThreads, 0, s>>>(
                x, static_cast<const int64_t*>(targets), logprob, entropy, lse, top_logprob, static_cast<int64_t*>(top_index), (int)d->vocab, d->ld_logits, d->scale, top_k);
        else
            token_logprob_kernel<T, int32_t><<<(unsigned)d->rows, kLogprobThreads, 0, s>>>(
                x, static_cast<const int32_t*>(targets), logprob, entropy, lse, top_logprob, static_cast<int32_t*>(top_index), (int)d->vocab, d->ld_logits, d->scale, top_k);
    });
    NZB_CUDA_TRY(cudaGetLastError());
    return NZB_OK;
}

int nzb_token_logprob_backward(const nzb_token_logprob_desc* d, const void* logits, const void* targets, const float* lse,
                               const float* entropy, const float* dlogprob, const float* dentropy, void* dlogits, void* stream) {
    int rc = check_logprob(d);
    if (rc != NZB_OK) return rc;
    if (d->ld_dlogits < d->vocab) return fail(NZB_ERR_BAD_ARG, "leading dimension smaller than the row length");
    if (d->rows == 0 || d->vocab == 0) return NZB_OK;
    if (!logits || !targets || !lse || !dlogits || (dentropy && !entropy))
        return fail(NZB_ERR_BAD_ARG, "logits, targets, lse, dlogits (and entropy beside dentropy) must be non-null");
    const int64_t size = dtype_size(d->dtype);
    if (!aligned_to(logits, size) || !aligned_to(dlogits, size)) return fail(NZB_ERR_BAD_ARG, "pointer is not a multiple of its element's size");
    DeviceState* ds;
    rc = get_device_state(&ds);
    if (rc != NZB_OK) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    NZB_DISPATCH_DTYPE(d->dtype, T, {
        const int64_t blocks = (d->vocab + Elem<T>::VEC - 1) / Elem<T>::VEC + 1;
        int64_t gx = (blocks + 1023) / 1024;
        for (int64_t r0 = 0; r0 < d->rows; r0 += 65535) {
            const int64_t n = d->rows - r0 < 65535 ? d->rows - r0 : 65535;
            const dim3 grid((unsigned)gx, (unsigned)n);
            const T* x = static_cast<const T*>(logits) + r0 * d->ld_logits;
            T* o = static_cast<T*>(dlogits) + r0 * d->ld_dlogits;
            const float* ent = dentropy ? entropy + r0 : nullptr;
            const float* dlp = dlogprob ? dlogprob + r0 : nullptr;
            const float* dent = dentropy ? dentropy + r0 : nullptr;
            if (d->index_type == NZB_I64)
                token_logprob_backward_kernel<T, int64_t><<<grid, 256, 0, s>>>(x, static_cast<const int64_t*>(targets) + r0, lse + r0, ent, dlp, dent, o, (int)d->vocab, d->ld_logits, d->ld_dlogits, d->scale);
            else
                token_logprob_backward_kernel<T, int32_t><<<grid, 256, 0, s>>>(x, static_cast<const int32_t*>(targets) + r0, lse + r0, ent, dlp, dent, o, (int)d->vocab, d->ld_logits, d->ld_dlogits, d->scale);
        }
    });
    NZB_CUDA_TRY(cudaGetLastError());
    return NZB_OK;
}

}  // extern "C"
