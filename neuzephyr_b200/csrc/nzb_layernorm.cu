// Layer norm over rows, forward and backward with the gradients of its two parameters.
//
// Forward: y = (x - mean) rstd gamma + beta. A row is read once and stays in registers: its mean first, then the
// variance of the centred values (no cancellation when the mean is large against the spread).
// Backward, h = (x - mean) rstd, g = dy gamma:
//   dx = rstd (g - mean(g) - h mean(g h)), dgamma = sum_rows dy h, dbeta = sum_rows dy.
// Every CTA walks many rows with each thread at the same columns, so the parameters' sums stay in registers
// and leave once per CTA; a second kernel adds the CTAs' sums in order (same bits every time).
// Rows that do not start on 16 bytes: the columns a thread owns shift with the row's address, with a period of
// at most 16 / element size rows, so a CTA takes rows of one residue only and its threads keep their columns.
#include <cooperative_groups.h>

#include "nzb_elem.cuh"
#include "nzb_internal.h"

namespace nzb {

namespace cg = cooperative_groups;

// Sum over the CTA, the same bits in every thread. buf: a float per warp, not written again before the next barrier.
__device__ __forceinline__ float block_sum(float v, float* buf) {
    v = warp_sum(v);
    const int warps = blockDim.x >> 5;
    if (warps == 1) return v;
    if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
    __syncthreads();
    const int lane = threadIdx.x & 31;
    return warp_sum(lane < warps ? buf[lane] : 0.f);
}

constexpr int kNormElems = 16;     // backward: columns per thread
// Backward: rows on their way.
constexpr int kNormStages = 3;
constexpr int kNormMaxCluster = 4;
// Forward: 32 elements a thread need 96 registers (with 80 the spilled ones cost 8191 x 5003 fp16 a tenth), 16 and fewer 64.
template <typename T, int ELEMS>
constexpr int norm_max_threads() { return ELEMS == 32 ? 640 : 1024; }
constexpr int kNormBackwardMaxThreads = 512;  // backward: 32 sums and the row's 32 factors per thread
constexpr int kNormSmem = 225 * 1024;          // dynamic shared memory of a CTA
constexpr int kNormLongParts = 64;
constexpr int kNormSms = 148;      // the workspace holds one pair of sums per CTA of a grid over this many SMs

// A thread's share of a row: the blocks t, t + nt, ... of VPT. The same for every row of a residue.
template <typename T, int VPT>
struct RowShare {
    static constexpr int VEC = Elem<T>::VEC;
    int first0, pitch;      // first element of block 0; elements between two blocks
    uint32_t some, whole;   // a bit per block: holds any of the row's elements; holds nothing else
    float extra;            // elements of its cut blocks that lie outside the row
    __device__ __forceinline__ RowShare(int t, int nt, int lead, int dim) : first0(t * VEC - lead), pitch(nt * VEC), some(0), whole(0) {
        int in = 0;
#pragma unroll
        for (int k = 0; k < VPT; k++) {
            if (first(k) < dim) some |= 1u << k;
            if (first(k) >= 0 && first(k) + VEC <= dim) whole |= 1u << k;
            in += max(0, min(first(k) + VEC, dim) - max(first(k), 0));
        }
        extra = static_cast<float>(__popc(some) * VEC - in);
    }
    __device__ __forceinline__ int first(int k) const { return first0 + k * pitch; }
    __device__ __forceinline__ bool has(int k) const { return some >> k & 1; }
    __device__ __forceinline__ float weight(int k) const { return has(k) ? 1.f : 0.f; }
    // every block of the warp's lies whole within the row
    __device__ __forceinline__ bool plain() const { return __all_sync(0xffffffffu, whole == (1u << VPT) - 1); }
    __device__ __forceinline__ float count() const { return __popc(some) * static_cast<float>(VEC) - extra; }
    // Gives the elements outside the row, in this thread's places in shared memory, the value of one inside it (so that
    // they deviate from the mean like any other and can be subtracted from the sums without loss), or zero; returns that
    // value. Only the threads at the row's ends have any, and nobody else pays for a mask.
    __device__ __forceinline__ float patch(uint4* ring, int nt, int dim, bool zero) const {
        if (extra == 0.f) return 0.f;
        T value = Elem<T>::from(0.f);
        for (int k = 0; k < VPT && !zero; k++)
            if (has(k) && !(whole >> k & 1)) value = reinterpret_cast<T*>(ring + k * nt)[max(0, -first(k))];
        for (int k = 0; k < VPT; k++)
            if (has(k) && !(whole >> k & 1))
                for (int i = 0; i < VEC; i++)
                    if (first(k) + i < 0 || first(k) + i >= dim) reinterpret_cast<T*>(ring + k * nt)[i] = value;
        return Elem<T>::to(value);
    }
    // Sum of f over the thread's elements of a row in memory.
    template <class F>
    __device__ __forceinline__ float sum(const T* row, int dim, F f) const {
        float s = 0.f;
#pragma unroll 1
        for (int e = 0; e < VPT * VEC; e++) {
            const int c = first(e / VEC) + e % VEC;
            if (c >= 0 && c < dim) s += f(Elem<T>::to(row[c]));
        }
        return s;
    }
    // Starts the copies of the row whose block 0 is `from` to this thread's own places in shared memory, nt blocks apart
    // (copies to places that are not side by side in a warp take half as long again); the same thread reads them after they have landed, so no barrier is needed. A block at the row's end brings elements of its
    // neighbours, or of the gap between two rows, along, which patch() replaces; only blocks that reach beyond the tensor
    // (of n elements from `base`) go element by element (waiting for them cost a memory latency per row).
    __device__ __forceinline__ void fetch(uint4* ring, int nt, const T* from, bool plain, bool border, const T* base, int64_t n) const {
        const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(ring));
        const auto copy = [&](int k) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + k * nt * 16), "l"(from + k * pitch) : "memory"); };
        if (plain) {
#pragma unroll
            for (int k = 0; k < VPT; k++) copy(k);
            return;
        }
#pragma unroll
        for (int k = 0; k < VPT; k++) {
            if (!has(k)) continue;
            const int64_t at = from - base + k * pitch;
            if (border && (at < 0 || at + VEC > n)) ring[k * nt] = load_block(base, at, n);
            else copy(k);
        }
    }
    // Writes block k of a row that starts on the same offset from 16 bytes; block0: where block 0 lies.
    __device__ __forceinline__ void store(T* block0, int k, bool plain, int dim, const float (&f)[VEC]) const {
        if (plain || (whole >> k & 1)) *reinterpret_cast<uint4*>(block0 + k * pitch) = Elem<T>::pack(f);
        else if (has(k)) store_block(block0 - first0, first(k), dim, Elem<T>::pack(f));
    }
};
// Rows at either end of a tensor whose blocks may reach beyond it: more than one when a block holds several rows.
__device__ __forceinline__ int border_rows(int64_t ld, int vec) { return ld < vec ? vec : 1; }
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

// A group of `nt` threads works on a row; the CTA's groups walk the rows of one residue, so that a thread's columns
// stay the same: gamma and beta lie in shared memory, all groups', thread by thread as they are read (read from memory
// unaligned for every row they cost more than the row: 8191 x 5003 fp16 113 us). A thread's are an odd number of 16-byte
// blocks: no bank conflicts, and addresses that differ by constants. STAGES rows per group are on their way while one is worked on. EXACT: rows start on 16 bytes and fill
// the group's threads, so nothing is masked.
// Statistics with one barrier: a warp's mean and its squares about that mean, then the warps' pairs joined,
// M2 = sum_w (M2_w + n_w (mean_w - mean)^2); no difference of large numbers anywhere.
template <typename T, int ELEMS, int STAGES, bool EXACT>
__global__ void __launch_bounds__(norm_max_threads<T, ELEMS>())
layernorm_kernel(const T* x, const float* __restrict__ gamma, const float* __restrict__ beta, T* y,
                 float* __restrict__ mean_out, float* __restrict__ rstd_out, int64_t rows, int dim, int64_t ld_x,
                 int64_t ld_y, float eps, int period, int y_together, int nt, int groups) {
    constexpr int VEC = Elem<T>::VEC, VPT = ELEMS / VEC, Q = ELEMS / 4;
    extern __shared__ uint4 smem_norm[];
    __shared__ float2 buf[2][32];  // per warp of the CTA: mean and M2
    const int group = threadIdx.x / nt, t = threadIdx.x - group * nt, lane = threadIdx.x & 31;
    const int warps = nt >> 5, warp0 = group * warps, warp = threadIdx.x >> 5;
    float4* params = reinterpret_cast<float4*>(smem_norm) + t * (2 * Q + 1);             // [nt][gamma, beta][Q], one unused
    uint4* ring = smem_norm + nt * (2 * Q + 1) + group * (STAGES * VPT * nt) + t;   // per group [STAGES][VPT][nt]
    const int residue = blockIdx.x % period;
    const int lead = EXACT ? 0 : row_lead(x + residue * ld_x);
    const int64_t span = (rows - 1) * ld_x + dim;
    const int edge = border_rows(ld_x, VEC);
    const int64_t step = static_cast<int64_t>(gridDim.x / period) * groups * period;
    const int64_t first_row = residue + static_cast<int64_t>(period) * (static_cast<int64_t>(blockIdx.x / period) * groups + group);
    const RowShare<T, VPT> share(t, nt, lead, dim);
    if (!EXACT) {
        // blocks beyond the row are read as zeros, with weight zero
#pragma unroll
        for (int k = 0; k < STAGES * VPT; k++)
            if (!share.has(k % VPT)) ring[k * nt] = make_uint4(0, 0, 0, 0);
    }
    const bool plain = EXACT || share.plain();
    const T* next = x + first_row * ld_x + share.first0;  // of the row to fetch next
    const int64_t step_x = step * ld_x, step_y = step * ld_y;
    const auto fetch = [&](int64_t r, int stage) {
        if (r < rows) share.fetch(ring + stage * VPT * nt, nt, next, plain, !EXACT && (r < edge || r >= rows - edge), x, span);
        next += step_x;
        copies_commit();
    };
#pragma unroll
    for (int s = 0; s < STAGES; s++) fetch(first_row + s * step, s);
    for (int q = group; q < Q; q += groups) {
        float g[4], b[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int e = q * 4 + i, c = (t + e / VEC * nt) * VEC - lead + e % VEC;
            const bool in = c >= 0 && c < dim;
            g[i] = in ? (gamma ? gamma[c] : 1.f) : 0.f;
            b[i] = in && beta ? beta[c] : 0.f;
        }
        params[q] = make_float4(g[0], g[1], g[2], g[3]);
        params[Q + q] = make_float4(b[0], b[1], b[2], b[3]);
    }
    __syncthreads();
    // elements of this warp and, lane by lane, of the group's warps
    const float n_warp = warp_sum(share.count()), inv_warp = n_warp > 0.f ? 1.f / n_warp : 0.f, inv = 1.f / dim;
    float n_lane = 0.f;
    if (warps > 1) {
        if (lane == 0) buf[0][warp].x = n_warp;
        __syncthreads();
        n_lane = lane < warps ? buf[0][warp0 + lane].x : 0.f;
        __syncthreads();
    }
    int turn = 0, stage = 0;
    T* yr = y + first_row * ld_y + share.first0;
    for (int64_t r = first_row; r < rows; r += step, turn ^= 1, yr += step_y) {
        copies_wait<STAGES - 1>();
        uint4* row = ring + stage * VPT * nt;
        const float extra_value = plain ? 0.f : share.patch(row, nt, dim, false);
        float2 v[VPT][VEC / 2];
        float sum = 0.f, sq = 0.f;
#pragma unroll
        for (int k = 0; k < VPT; k++) {
            float f[VEC];
            Elem<T>::unpack(row[k * nt], f);
            float2 part = make_float2(0.f, 0.f);
#pragma unroll
            for (int i = 0; i < VEC / 2; i++) {
                v[k][i] = make_float2(f[2 * i], f[2 * i + 1]);
                part = add2(part, v[k][i]);
            }
            sum += part.x + part.y;
        }
        if (!plain) sum = fmaf(-share.extra, extra_value, sum);
        fetch(r + STAGES * step, stage);
        stage = stage + 1 == STAGES ? 0 : stage + 1;
        float mean = warp_sum(sum) * inv_warp;
        const float2 minus = make_float2(-mean, -mean);
#pragma unroll
        for (int k = 0; k < VPT; k++) {
            float2 part = make_float2(0.f, 0.f);
#pragma unroll
            for (int i = 0; i < VEC / 2; i++) {
                const float2 d = add2(v[k][i], minus);
                part = fma2(d, d, part);
            }
            sq = plain ? sq + (part.x + part.y) : fmaf(share.weight(k), part.x + part.y, sq);
        }
        if (!plain) {
            const float d = extra_value - mean;
            sq = fmaf(-share.extra * d, d, sq);
        }
        float m2 = warp_sum(sq);
        if (!plain && !(m2 < INFINITY)) {
            // what is subtracted or weighted by 0 above may have left fp32's range where the row's own elements do not: their
            // sums again, without any other (a mask for every row would cost 8191 x 5003 fp16 two microseconds)
            mean = warp_sum(share.sum(x + r * ld_x, dim, [](float f) { return f; })) * inv_warp;
            m2 = warp_sum(share.sum(x + r * ld_x, dim, [&](float f) { return (f - mean) * (f - mean); }));
        }
        if (warps > 1) {
            if (lane == 0) buf[turn][warp] = make_float2(mean, m2);
            asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(nt) : "memory");
            const float2 part = lane < warps ? buf[turn][warp0 + lane] : make_float2(0.f, 0.f);
            mean = warp_sum(part.x * n_lane) * inv;
            const float d = part.x - mean;
            m2 = warp_sum(lane < warps ? fmaf(n_lane * d, d, part.y) : 0.f);
        }
        const float rstd = rsqrtf(fmaf(m2, inv, eps));
        if (t == 0) {
            if (mean_out) mean_out[r] = mean;
            if (rstd_out) rstd_out[r] = rstd;
        }
        const float2 rs = make_float2(rstd, rstd), shift = make_float2(-mean, -mean);
#pragma unroll
        for (int k = 0; k < VPT; k++) {
            if (!plain && !share.has(k)) continue;
            float o[VEC];
#pragma unroll
            for (int q = 0; q < VEC / 4; q++) {
                const float4 g = params[k * (VEC / 4) + q], b = params[Q + k * (VEC / 4) + q];
                // (x - mean) rstd, then gamma and beta
                const float2 lo = fma2(mul2(add2(v[k][2 * q], shift), rs), make_float2(g.x, g.y), make_float2(b.x, b.y));
                const float2 hi = fma2(mul2(add2(v[k][2 * q + 1], shift), rs), make_float2(g.z, g.w), make_float2(b.z, b.w));
                o[4 * q] = lo.x; o[4 * q + 1] = lo.y; o[4 * q + 2] = hi.x; o[4 * q + 3] = hi.y;
            }
            if (EXACT || y_together) {
                share.store(yr, k, plain, dim, o);
            } else {
#pragma unroll
                for (int i = 0; i < VEC; i++) {
                    const int c = share.first(k) + i;
                    if (c >= 0 && c < dim) yr[c - share.first0] = Elem<T>::from(o[i]);
                }
            }
        }
    }
    copies_wait<0>();
}

// Rows too long for the registers of a CTA: three walks over the row.
template <typename T>
__global__ void __launch_bounds__(1024)
layernorm_long_kernel(const T* x, const float* __restrict__ gamma, const float* __restrict__ beta, T* y,
                      float* __restrict__ mean_out, float* __restrict__ rstd_out, int dim, int64_t ld_x, int64_t ld_y, float eps) {
    __shared__ float buf[2][32];
    const int64_t r = blockIdx.x;
    const T* xr = x + r * ld_x;
    T* yr = y + r * ld_y;
    float sum = 0.f;
    for (int c = threadIdx.x; c < dim; c += 1024) sum += Elem<T>::to(xr[c]);
    const float mean = block_sum(sum, buf[0]) / dim;
    float sq = 0.f;
    for (int c = threadIdx.x; c < dim; c += 1024) {
        const float d = Elem<T>::to(xr[c]) - mean;
        sq += d * d;
    }
    const float rstd = 1.f / sqrtf(block_sum(sq, buf[1]) / dim + eps);
    if (threadIdx.x == 0) {
        if (mean_out) mean_out[r] = mean;
        if (rstd_out) rstd_out[r] = rstd;
    }
    for (int c = threadIdx.x; c < dim; c += 1024)
        yr[c] = Elem<T>::from((Elem<T>::to(xr[c]) - mean) * rstd * (gamma ? gamma[c] : 1.f) + (beta ? beta[c] : 0.f));
}

// Two sums over the warp in one chain of shuffles: the lower half of the lanes ends with the first, the upper half with
// the second.
__device__ __forceinline__ float warp_sum_two(float a, float b, int lane) {
    const bool upper = lane & 16;
    float v = (upper ? b : a) + __shfl_xor_sync(0xffffffffu, upper ? a : b, 16);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// The same walk as the forward kernel's, x and dy on their way together. Every group keeps its sums of the parameters'
// gradients; at the end the CTA adds its groups', in order. CLUSTER: rows of more than 8192 elements, in as many
// parts of `share_cols` columns as the cluster has CTAs; the parts' two sums meet in everybody's shared memory, with the
// cluster's barrier in place of the CTA's.
template <typename T, bool EXACT, bool CLUSTER>
__global__ void __launch_bounds__(kNormBackwardMaxThreads)
layernorm_backward_kernel(const T* dy, const T* x, const float* __restrict__ mean, const float* __restrict__ rstd,
                          const float* __restrict__ gamma, T* dx, float* __restrict__ partial, int64_t rows, int row_dim,
                          int64_t ld_x, int64_t ld_dy, int64_t ld_dx, int period, int add_dx, int nt, int groups, int cluster,
                          int share_cols) {
    constexpr int VEC = Elem<T>::VEC, VPT = kNormElems / VEC, Q = kNormElems / 4, STAGES = kNormStages;
    extern __shared__ uint4 smem_norm[];
    __shared__ float buf[2][2][kNormMaxCluster * 16];  // [turn][sum][warp of the CTA, of the cluster]
    const int group = threadIdx.x / nt, t = threadIdx.x - group * nt, lane = threadIdx.x & 31;
    const int warps = nt >> 5, warp0 = group * warps, warp = threadIdx.x >> 5;
    float4* params = reinterpret_cast<float4*>(smem_norm) + t * (Q | 1);                   // [nt][Q], all groups'
    uint4* ring = smem_norm + (Q | 1) * nt + group * (STAGES * 2 * VPT * nt) + t;          // per group [stage][x, dy][VPT][nt]
    // this CTA's columns, as a matrix of its own
    const int part = CLUSTER ? blockIdx.x % cluster : 0, c0 = part * share_cols;
    const int64_t walker = CLUSTER ? blockIdx.x / cluster : blockIdx.x, walkers = CLUSTER ? gridDim.x / cluster : gridDim.x;
    const int dim = CLUSTER ? min(share_cols, row_dim - c0) : row_dim;
    if (CLUSTER) {
        x += c0;
        dy += c0;
        if (dx) dx += c0;
        if (gamma) gamma += c0;
    }
    const int residue = static_cast<int>(walker % period);
    const int lead = EXACT ? 0 : row_lead(x + residue * ld_x);
    const int64_t span_x = (rows - 1) * ld_x + dim, span_dy = (rows - 1) * ld_dy + dim;
    const int edge = border_rows(min(ld_x, ld_dy), VEC);
    const int64_t step = walkers / period * groups * period;
    const int64_t first_row = residue + period * (walker / period * groups + group);
    const RowShare<T, VPT> share(t, nt, lead, dim);
    if (!EXACT) {
        // blocks beyond the row are read as zeros: a dy of zero adds nothing
#pragma unroll
        for (int k = 0; k < STAGES * 2 * VPT; k++)
            if (!share.has(k % VPT)) ring[k * nt] = make_uint4(0, 0, 0, 0);
    }
    const bool plain = EXACT || share.plain();
    const T* next_x = x + first_row * ld_x + share.first0;  // of the row to fetch next
    const T* next_dy = dy + first_row * ld_dy + share.first0;
    const int64_t step_x = step * ld_x, step_dy = step * ld_dy, step_dx = step * ld_dx;
    const auto fetch = [&](int64_t r, int stage) {
        if (r < rows) {
            const bool border = !EXACT && (r < edge || r >= rows - edge);
            share.fetch(ring + stage * 2 * VPT * nt, nt, next_x, plain, border, x, span_x);
            share.fetch(ring + (stage * 2 + 1) * VPT * nt, nt, next_dy, plain, border, dy, span_dy);
        }
        next_x += step_x;
        next_dy += step_dy;
        copies_commit();
    };
#pragma unroll
    for (int s = 0; s < STAGES; s++) fetch(first_row + s * step, s);
    float2 dg[VPT][VEC / 2], db[VPT][VEC / 2];
#pragma unroll
    for (int k = 0; k < VPT; k++)
#pragma unroll
        for (int i = 0; i < VEC / 2; i++) dg[k][i] = db[k][i] = make_float2(0.f, 0.f);
    for (int q = group; q < Q; q += groups) {
        float g[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int e = q * 4 + i, c = (t + e / VEC * nt) * VEC - lead + e % VEC;
            g[i] = c >= 0 && c < dim ? (gamma ? gamma[c] : 1.f) : 0.f;
        }
        params[q] = make_float4(g[0], g[1], g[2], g[3]);
    }
    __syncthreads();
    if (CLUSTER) cg::this_cluster().sync();  // everybody runs before anybody writes into another's shared memory
    const float inv = 1.f / row_dim;
    int turn = 0, stage = 0;
    float next_mean = first_row < rows ? mean[first_row] : 0.f, next_rstd = first_row < rows ? rstd[first_row] : 0.f;
    T* dxr = dx + first_row * ld_dx + share.first0;
    for (int64_t r = first_row; r < rows; r += step, turn ^= 1, dxr += step_dx) {
        const float2 rs = make_float2(next_rstd, next_rstd), minus = make_float2(-next_mean, -next_mean);
        if (r + step < rows) {
            next_mean = mean[r + step];
            next_rstd = rstd[r + step];
        }
        copies_wait<STAGES - 1>();
        uint4* xs = ring + stage * 2 * VPT * nt;
        uint4* ds = xs + VPT * nt;
        if (!plain) {
            // outside the row: an x of the row, whose h is finite where the row's are, and a dy of zero, which adds nothing
            share.patch(xs, nt, dim, false);
            share.patch(ds, nt, dim, true);
        }
        float2 h[VPT][VEC / 2], g[VPT][VEC / 2];
        float2 sg = make_float2(0.f, 0.f), sgh = sg;
#pragma unroll
        for (int k = 0; k < VPT; k++) {
            float fx[VEC], fd[VEC];
            Elem<T>::unpack(xs[k * nt], fx);
            Elem<T>::unpack(ds[k * nt], fd);
            // a place without elements: x is 0, and so has to be the mean, whose product with rstd may be inf (and its with 0 NaN)
            const float2 shift = plain || share.has(k) ? minus : make_float2(0.f, 0.f);
#pragma unroll
            for (int i = 0; i < VEC / 2; i++) {
                const float4 ga = params[k * (VEC / 4) + i / 2];
                const float2 d = make_float2(fd[2 * i], fd[2 * i + 1]);
                h[k][i] = mul2(add2(make_float2(fx[2 * i], fx[2 * i + 1]), shift), rs);
                g[k][i] = mul2(d, i & 1 ? make_float2(ga.z, ga.w) : make_float2(ga.x, ga.y));
                sg = add2(sg, g[k][i]);
                sgh = fma2(g[k][i], h[k][i], sgh);
                dg[k][i] = fma2(d, h[k][i], dg[k][i]);
                db[k][i] = add2(db[k][i], d);
            }
        }
        fetch(r + STAGES * step, stage);
        stage = stage + 1 == STAGES ? 0 : stage + 1;
        if (dx) {
            float s = warp_sum_two(sg.x + sg.y, sgh.x + sgh.y, lane);
            if (CLUSTER) {
                cg::cluster_group all = cg::this_cluster();
                if ((lane & 15) == 0)
                    for (int o = 0; o < cluster; o++) *all.map_shared_rank(&buf[turn][lane >> 4][part * warps + warp], o) = s;
                all.sync();  // the other turn's sums are not written again before everybody has passed
                s = 0.f;
                for (int w = lane & 15; w < cluster * warps; w += 16) s += buf[turn][lane >> 4][w];
            } else if (warps > 1) {
                if ((lane & 15) == 0) buf[turn][lane >> 4][warp] = s;
                asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(nt) : "memory");
                s = (lane & 15) < warps ? buf[turn][lane >> 4][warp0 + (lane & 15)] : 0.f;
            }
            if (CLUSTER || warps > 1) {
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
            }
            // dx = rstd (g - mean g - h mean(g h))
            s *= -rs.x * inv;
            const float other = __shfl_xor_sync(0xffffffffu, s, 16);
            const float m0 = lane & 16 ? other : s, m1 = lane & 16 ? s : other;
            const float2 m0s = make_float2(m0, m0), m1s = make_float2(m1, m1);
#pragma unroll
            for (int k = 0; k < VPT; k++) {
                if (!plain && !share.has(k)) continue;
                float o[VEC];
#pragma unroll
                for (int i = 0; i < VEC / 2; i++) {
                    const float2 d = fma2(g[k][i], rs, fma2(h[k][i], m1s, m0s));
                    o[2 * i] = d.x;
                    o[2 * i + 1] = d.y;
                }
                if (add_dx) {
                    float old[VEC];
                    Elem<T>::unpack(load_block(dxr - share.first0, share.first(k), dim), old);
#pragma unroll
                    for (int i = 0; i < VEC; i++) o[i] += old[i];
                }
                share.store(dxr, k, plain, dim, o);
            }
        }
    }
    copies_wait<0>();
    if (CLUSTER) cg::this_cluster().sync();  // nobody leaves while another CTA may still write its sums here
    if (!partial) return;
    if (groups > 1) {
        // every group's sums where its rows were, then group 0 adds them
        __syncthreads();
        float2* mine = reinterpret_cast<float2*>(ring - t) + t;  // [2 kNormElems / 2][nt]
        static_assert(STAGES * 2 * VPT * 16 >= 2 * kNormElems * 4, "the sums fit in the ring");
#pragma unroll
        for (int k = 0; k < VPT; k++)
#pragma unroll
            for (int i = 0; i < VEC / 2; i++) {
                mine[(k * (VEC / 2) + i) * nt] = dg[k][i];
                mine[(kNormElems / 2 + k * (VEC / 2) + i) * nt] = db[k][i];
            }
        __syncthreads();
        if (group) return;
        for (int o = 1; o < groups; o++) {
            const float2* theirs = mine + o * (STAGES * 2 * VPT * nt) * 2;
#pragma unroll
            for (int k = 0; k < VPT; k++)
#pragma unroll
                for (int i = 0; i < VEC / 2; i++) {
                    dg[k][i] = add2(dg[k][i], theirs[(k * (VEC / 2) + i) * nt]);
                    db[k][i] = add2(db[k][i], theirs[(kNormElems / 2 + k * (VEC / 2) + i) * nt]);
                }
        }
    }
    float* pg = partial + walker * 2 * row_dim + c0;
#pragma unroll
    for (int k = 0; k < VPT; k++) {
#pragma unroll
        for (int i = 0; i < VEC; i++) {
            const int c = share.first(k) + i;
            if (c >= 0 && c < dim) {
                pg[c] = i & 1 ? dg[k][i / 2].y : dg[k][i / 2].x;
                pg[row_dim + c] = i & 1 ? db[k][i / 2].y : db[k][i / 2].x;
            }
        }
    }
}

// Rows longer than the fused kernel's, or tensors whose rows start at different offsets: one CTA per row for dx,
// and a kernel of its own for the parameters.
template <typename T>
__global__ void __launch_bounds__(512)
layernorm_dx_kernel(const T* dy, const T* x, const float* __restrict__ mean, const float* __restrict__ rstd,
                    const float* __restrict__ gamma, T* dx, int dim, int64_t ld_x, int64_t ld_dy, int64_t ld_dx, int add_dx) {
    __shared__ float buf[2][32];
    const int64_t r = blockIdx.x;
    const T* xr = x + r * ld_x;
    const T* dyr = dy + r * ld_dy;
    T* dxr = dx + r * ld_dx;
    const float mu = mean[r], rs = rstd[r];
    float sg = 0.f, sgh = 0.f;
    for (int c = threadIdx.x; c < dim; c += 512) {
        const float g = Elem<T>::to(dyr[c]) * (gamma ? gamma[c] : 1.f);
        sg += g;
        sgh += g * ((Elem<T>::to(xr[c]) - mu) * rs);
    }
    sg = block_sum(sg, buf[0]) / dim;
    sgh = block_sum(sgh, buf[1]) / dim;
    for (int c = threadIdx.x; c < dim; c += 512) {
        const float g = Elem<T>::to(dyr[c]) * (gamma ? gamma[c] : 1.f);
        float d = rs * (g - sg - (Elem<T>::to(xr[c]) - mu) * rs * sgh);
        if (add_dx) d += Elem<T>::to(dxr[c]);
        dxr[c] = Elem<T>::from(d);
    }
}
template <typename T>
__global__ void __launch_bounds__(256)
layernorm_dparams_kernel(const T* __restrict__ dy, const T* __restrict__ x, const float* __restrict__ mean,
                         const float* __restrict__ rstd, float* __restrict__ partial, int64_t rows, int dim, int64_t ld_x,
                         int64_t ld_dy) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= dim) return;
    const int64_t r0 = rows * blockIdx.y / gridDim.y, r1 = rows * (blockIdx.y + 1) / gridDim.y;
    float dg = 0.f, db = 0.f;
#pragma unroll 4
    for (int64_t r = r0; r < r1; r++) {
        const float d = Elem<T>::to(dy[r * ld_dy + c]);
        db += d;
        dg += d * ((Elem<T>::to(x[r * ld_x + c]) - mean[r]) * rstd[r]);
    }
    partial[static_cast<int64_t>(blockIdx.y) * 2 * dim + c] = dg;
    partial[static_cast<int64_t>(blockIdx.y) * 2 * dim + dim + c] = db;
}

// Adds the CTAs' sums: 32 columns x 8 slices of the CTAs per block.
__global__ void __launch_bounds__(256)
layernorm_reduce_kernel(const float* __restrict__ partial, int parts, float* __restrict__ dgamma, float* __restrict__ dbeta,
                        int dim, int overwrite) {
    __shared__ float buf[8][32];
    const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;  // over both parameters
    float s = 0.f;
    if (c < 2 * dim) {
        const int p1 = parts * (slice + 1) / 8;
#pragma unroll 8
        for (int p = parts * slice / 8; p < p1; p++) s += partial[static_cast<int64_t>(p) * 2 * dim + c];
    }
    buf[slice][lane] = s;
    __syncthreads();
    if (slice || c >= 2 * dim) return;
#pragma unroll
    for (int i = 1; i < 8; i++) s += buf[i][lane];
    float* to = c < dim ? dgamma : dbeta;
    if (!to) return;
    to += c < dim ? c : c - dim;
    *to = overwrite ? s : *to + s;
}

static int check_layernorm(const nzb_layernorm_desc* d) {
    if (!d) return fail(NZB_ERR_BAD_ARG, "descriptor is null");
    if (d->rows < 0 || d->dim < 0) return fail(NZB_ERR_BAD_ARG, "negative extent");
    if (d->dim > (1 << 24) || d->rows > INT32_MAX) return fail(NZB_ERR_UNSUPPORTED, "dim at most 2^24, rows below 2^31");
    if (!known_dtype(d->dtype)) return fail(NZB_ERR_BAD_ARG, "unknown element type");
    if (d->ld_x < d->dim || d->ld_y < d->dim) return fail(NZB_ERR_BAD_ARG, "leading dimension smaller than the row length");
    if (!(d->eps >= 0.f)) return fail(NZB_ERR_BAD_ARG, "eps is negative or NaN");
    return NZB_OK;
}

static bool overlap(const float* a, const float* b, int64_t n) { return a && b && a < b + n && b < a + n; }

// Threads that hold a row of `dim` elements in registers, `elems` each; 0: more than `most`. lead: elements the row's
// first block may share with what is before it.
static int norm_threads(int64_t dim, int lead, int most, int elems) {
    const int64_t nt = round_up((dim + lead + elems - 1) / elems, 32);
    return nt <= most ? (int)nt : 0;
}
// CTAs of the backward kernels, at most: one for each SM, and one per residue at least; 64 of the kernel that takes the
// longest rows, so that its workspace stays small beside them.
static int64_t norm_parts(const nzb_layernorm_desc* d) {
    const int64_t most = d->dim > (int64_t)kNormMaxCluster * kNormBackwardMaxThreads * kNormElems ? kNormLongParts : kNormSms;
    const int64_t ctas = d->rows < most ? d->rows : most;
    return ctas < 8 ? 8 : ctas;
}

template <typename T, bool CLUSTER>
static int launch_norm_backward(const nzb_layernorm_desc* d, const void* dy, const void* x, const float* mean, const float* rstd,
                                const float* gamma, void* dx, float* partial, int period, bool exact, int nt, int cluster,
                                int64_t share_cols, int64_t* parts, cudaStream_t s) {
    constexpr int ring = kNormStages * 2 * (int)(kNormElems / Elem<T>::VEC) * 16, params = ((kNormElems / 4) | 1) * 16;
    // as many groups as threads, named barriers, shared memory and rows allow (eight rows a group, to be worth its sums)
    int64_t groups = CLUSTER ? 1 : kNormBackwardMaxThreads / nt;
    const int64_t fit = (kNormSmem / nt - params) / ring, spread = (d->rows + 8 * kNormSms - 1) / (8 * kNormSms);
    if (groups > 15 && nt > 32) groups = 15;
    if (groups > fit) groups = fit;
    if (groups > spread) groups = spread;
    if (groups < 1) return fail(NZB_ERR_UNSUPPORTED, "a group's rows exceed shared memory");
    int64_t walkers = (d->rows + groups - 1) / groups;
    if (walkers > *parts / cluster) walkers = *parts / cluster;
    walkers = walkers / period * period;
    if (walkers == 0) walkers = period;
    *parts = walkers;
    const auto kernel = exact ? layernorm_backward_kernel<T, true, CLUSTER> : layernorm_backward_kernel<T, false, CLUSTER>;
    static std::atomic<uint64_t> smem_set[2];
    int rc = ensure_dynamic_smem(smem_set[exact], reinterpret_cast<const void*>(kernel), kNormSmem);
    if (rc != NZB_OK) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(walkers * cluster));
    cfg.blockDim = dim3((unsigned)(groups * nt));
    cfg.dynamicSmemBytes = (size_t)(nt * (params + groups * ring));
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = CLUSTER ? 1 : 0;
    NZB_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, static_cast<const T*>(dy), static_cast<const T*>(x), mean, rstd, gamma,
                                    static_cast<T*>(dx), partial, d->rows, (int)d->dim, d->ld_x, d->ld_y, d->ld_dx, period,
                                    (int)!d->overwrite_dx, nt, (int)groups, cluster, (int)share_cols));
    return NZB_OK;
}

}  // namespace nzb

using namespace nzb;

extern "C" {

int nzb_layernorm_forward(const nzb_layernorm_desc* d, const void* x, const float* gamma, const float* beta, void* y,
                          float* mean, float* rstd, void* stream) {
    int rc = check_layernorm(d);
    if (rc != NZB_OK) return rc;
    if (d->rows == 0) return NZB_OK;
    if (overlap(mean, rstd, d->rows)) return fail(NZB_ERR_BAD_ARG, "mean and rstd overlap");
    if (d->dim == 0) {  // the mean of nothing: every bit set is a NaN
        if (mean) NZB_CUDA_TRY(cudaMemsetAsync(mean, 0xff, (size_t)d->rows * 4, static_cast<cudaStream_t>(stream)));
        if (rstd) NZB_CUDA_TRY(cudaMemsetAsync(rstd, 0xff, (size_t)d->rows * 4, static_cast<cudaStream_t>(stream)));
        return NZB_OK;
    }
    if (!x || !y) return fail(NZB_ERR_BAD_ARG, "x and y must be non-null");
    if (x == y && d->ld_x != d->ld_y) return fail(NZB_ERR_BAD_ARG, "y in place of x needs its leading dimension");
    const int64_t size = dtype_size(d->dtype);
    if (!aligned_to(x, size) || !aligned_to(y, size)) return fail(NZB_ERR_BAD_ARG, "pointer is not a multiple of its element's size");
    DeviceState* ds;
    rc = get_device_state(&ds);
    if (rc != NZB_OK) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    NZB_DISPATCH_DTYPE(d->dtype, T, {
        constexpr int VEC = Elem<T>::VEC;
        const bool repeats = d->ld_x * size % 16 == 0;
        const int period = repeats ? 1 : VEC;
        // four blocks per thread: the instructions of the sums' joins are per thread
        constexpr int WIDE = VEC * 4;
        const int lead = repeats && aligned_to(x, 16) ? 0 : VEC - 1;
        // rows for less than one round of the SMs: one block per thread shortens a row's way (64 x 1024 fp32: 2.8 us
        // instead of 4.2)
        int nt = d->rows <= ds->sm_count ? norm_threads(d->dim, lead, 1024, VEC) : 0;
        const bool y_together = reinterpret_cast<uintptr_t>(x) % 16 == reinterpret_cast<uintptr_t>(y) % 16 && d->ld_x * size % 16 == d->ld_y * size % 16;
        const int elems = nt ? VEC : WIDE, most = nt ? 1024 : norm_max_threads<T, WIDE>();
        if (!nt) nt = norm_threads(d->dim, lead, most, elems);
        const int params = nt * (elems / 2 + 1) * 16, row = nt * elems / VEC * 16;
        const int stages = elems == VEC || params + 2 * row > kNormSmem ? 1 : 2;
        const T* xp = static_cast<const T*>(x);
        T* yp = static_cast<T*>(y);
        if (nt && params + stages * row <= kNormSmem) {
            const bool exact = lead == 0 && d->dim == (int64_t)nt * elems && y_together;
            // as many groups as threads, named barriers (of groups of several warps), shared memory and rows allow
            int64_t groups = most / nt;
            const int64_t fit = (kNormSmem - params) / (stages * row), spread = (d->rows + ds->sm_count - 1) / ds->sm_count;
            if (groups > 15 && nt > 32) groups = 15;
            if (groups > fit) groups = fit;
            if (groups > spread) groups = spread;
            int64_t ctas = (d->rows + groups - 1) / groups;
            if (ctas > ds->sm_count) ctas = ds->sm_count;
            ctas = ctas / period * period;
            if (ctas == 0) ctas = period;
            const auto kernel = elems == VEC ? (exact ? layernorm_kernel<T, VEC, 1, true> : layernorm_kernel<T, VEC, 1, false>)
                                : stages == 1 ? (exact ? layernorm_kernel<T, WIDE, 1, true> : layernorm_kernel<T, WIDE, 1, false>)
                                              : (exact ? layernorm_kernel<T, WIDE, 2, true> : layernorm_kernel<T, WIDE, 2, false>);
            static std::atomic<uint64_t> smem_set[6];
            rc = ensure_dynamic_smem(smem_set[(elems == VEC ? 0 : 2 * stages) + exact], reinterpret_cast<const void*>(kernel), kNormSmem);
            if (rc != NZB_OK) return rc;
            kernel<<<(unsigned)ctas, (unsigned)(groups * nt), (size_t)(params + groups * stages * row), s>>>(
                xp, gamma, beta, yp, mean, rstd, d->rows, (int)d->dim, d->ld_x, d->ld_y, d->eps, period, y_together, nt, (int)groups);
        } else {
            layernorm_long_kernel<T><<<(unsigned)d->rows, 1024, 0, s>>>(xp, gamma, beta, yp, mean, rstd, (int)d->dim, d->ld_x, d->ld_y, d->eps);
        }
    });
    NZB_CUDA_TRY(cudaGetLastError());
    return NZB_OK;
}

int nzb_layernorm_backward_workspace_bytes(const nzb_layernorm_desc* d, size_t* bytes_out) {
    if (!bytes_out) return fail(NZB_ERR_BAD_ARG, "bytes_out is null");
    int rc = check_layernorm(d);
    if (rc != NZB_OK) return rc;
    *bytes_out = (size_t)round_up(norm_parts(d) * 2 * d->dim * 4, 256);
    return NZB_OK;
}

int nzb_layernorm_backward(const nzb_layernorm_desc* d, const void* dy, const void* x, const float* mean, const float* rstd,
                           const float* gamma, void* dx, float* dgamma, float* dbeta, void* workspace,
                           size_t workspace_bytes, void* stream) {
    int rc = check_layernorm(d);
    if (rc != NZB_OK) return rc;
    const bool params = dgamma || dbeta;
    if (d->dim == 0 || (!dx && !params)) return NZB_OK;
    if (dx && d->ld_dx < d->dim) return fail(NZB_ERR_BAD_ARG, "leading dimension smaller than the row length");
    if (dx && ((dx == dy && d->ld_dx != d->ld_y) || (dx == x && d->ld_dx != d->ld_x)))
        return fail(NZB_ERR_BAD_ARG, "dx in place of dy or x needs its leading dimension");
    // both sums would go to one place, from different threads
    if (overlap(dgamma, dbeta, d->dim)) return fail(NZB_ERR_BAD_ARG, "dgamma and dbeta overlap");
    DeviceState* ds;
    rc = get_device_state(&ds);
    if (rc != NZB_OK) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (d->rows == 0) {  // sums over no rows
        if (d->overwrite_dparams && dgamma) NZB_CUDA_TRY(cudaMemsetAsync(dgamma, 0, (size_t)d->dim * 4, s));
        if (d->overwrite_dparams && dbeta) NZB_CUDA_TRY(cudaMemsetAsync(dbeta, 0, (size_t)d->dim * 4, s));
        return NZB_OK;
    }
    if (!dy || !x || !mean || !rstd) return fail(NZB_ERR_BAD_ARG, "dy, x, mean and rstd must be non-null");
    const int64_t size = dtype_size(d->dtype);
    if (!aligned_to(x, size) || !aligned_to(dy, size) || !aligned_to(dx, size))
        return fail(NZB_ERR_BAD_ARG, "pointer is not a multiple of its element's size");
    size_t need = 0;
    rc = nzb_layernorm_backward_workspace_bytes(d, &need);
    if (rc != NZB_OK) return rc;
    if (params && (!workspace || workspace_bytes < need))
        return fail(NZB_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", need, workspace ? workspace_bytes : (size_t)0);
    if (params && !aligned_to(workspace, 256)) return fail(NZB_ERR_WORKSPACE, "workspace must be 256-byte aligned");
    float* partial = params ? static_cast<float*>(workspace) : nullptr;
    int64_t parts = norm_parts(d);
    // the fused kernel needs the rows of all three tensors to start at the same offset from 16 bytes
    const auto offset = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16; };
    const bool together = offset(x) == offset(dy) && d->ld_x * size % 16 == d->ld_y * size % 16 &&
                          (!dx || (offset(x) == offset(dx) && d->ld_x * size % 16 == d->ld_dx * size % 16));
    const int period = d->ld_x * size % 16 == 0 ? 1 : (int)(16 / size);
    const int lead = period == 1 && aligned_to(x, 16) ? 0 : (int)(16 / size) - 1;
    // CTAs to a row, and the columns of each: whole blocks of 16 bytes. Shared memory holds the rows of 480 threads in fp32
    const int most = size == 4 ? kNormBackwardMaxThreads - 32 : kNormBackwardMaxThreads;
    int cluster = 1, nt = 0;
    int64_t share_cols = d->dim;
    for (; together && cluster <= kNormMaxCluster; cluster *= 2) {
        share_cols = cluster == 1 ? d->dim : round_up((d->dim + cluster - 1) / cluster, 16 / size);
        if ((nt = norm_threads(share_cols, lead, most, kNormElems)) != 0) break;
    }
    if (nt) {
        const bool exact = period == 1 && lead == 0 && share_cols == (int64_t)nt * kNormElems && share_cols * cluster == d->dim;
        NZB_DISPATCH_DTYPE(d->dtype, T, {
            rc = cluster == 1 ? launch_norm_backward<T, false>(d, dy, x, mean, rstd, gamma, dx, partial, period, exact, nt, 1, share_cols, &parts, s)
                              : launch_norm_backward<T, true>(d, dy, x, mean, rstd, gamma, dx, partial, period, exact, nt, cluster, share_cols, &parts, s);
        });
        if (rc != NZB_OK) return rc;
    } else {
        NZB_DISPATCH_DTYPE(d->dtype, T, {
            const T* xp = static_cast<const T*>(x);
            const T* dyp = static_cast<const T*>(dy);
            if (params) {
                if (parts > kNormLongParts) parts = kNormLongParts;
                const dim3 grid((unsigned)((d->dim + 255) / 256), (unsigned)parts);
                layernorm_dparams_kernel<T><<<grid, 256, 0, s>>>(dyp, xp, mean, rstd, partial, d->rows, (int)d->dim, d->ld_x, d->ld_y);
            }
            if (dx)
                layernorm_dx_kernel<T><<<(unsigned)d->rows, 512, 0, s>>>(dyp, xp, mean, rstd, gamma, static_cast<T*>(dx), (int)d->dim, d->ld_x, d->ld_y, d->ld_dx, !d->overwrite_dx);
        });
    }
    NZB_CUDA_TRY(cudaGetLastError());
    if (params) {
        layernorm_reduce_kernel<<<(unsigned)((2 * d->dim + 31) / 32), 256, 0, s>>>(partial, (int)parts, dgamma, dbeta, (int)d->dim, d->overwrite_dparams);
        NZB_CUDA_TRY(cudaGetLastError());
    }
    return NZB_OK;
}

}  // extern "C"
