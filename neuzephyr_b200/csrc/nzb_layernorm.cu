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
#include "nzb_internal.h"
#include "nzb_elem.cuh"

namespace nzb {

template <int WARPS>
__device__ __forceinline__ float block_sum(float v, float* buf) {
    v = warp_sum(v);
    if (WARPS == 1) return v;
    if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
    __syncthreads();
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < WARPS; i++) t += buf[i];
    return t;
}

// NT threads per row; a warp per row (eight rows per CTA) when NT == 32.
template <typename T, int NT, int VPT>
__global__ void __launch_bounds__(NT == 32 ? 256 : NT)
layernorm_kernel(const T* x, const float* __restrict__ gamma, const float* __restrict__ beta, T* y,
                 float* __restrict__ mean_out, float* __restrict__ rstd_out, int64_t rows, int dim, int64_t ld_x,
                 int64_t ld_y, float eps) {
    constexpr int VEC = Elem<T>::VEC, WARPS = NT / 32;
    __shared__ float buf[2][WARPS];
    const int t = NT == 32 ? threadIdx.x & 31 : threadIdx.x;
    const int64_t r = NT == 32 ? static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5) : blockIdx.x;
    if (r >= rows) return;
    const T* xr = x + r * ld_x;
    T* yr = y + r * ld_y;
    const int lead = row_lead(xr);
    float v[VPT][VEC];
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < VPT; k++) {
        const int first = (t + k * NT) * VEC - lead;
        uint4 u = make_uint4(0, 0, 0, 0);
        if (first < dim) u = load_block(xr, first, dim);
        Elem<T>::unpack(u, v[k]);
#pragma unroll
        for (int i = 0; i < VEC; i++) sum += v[k][i];
    }
    const float mean = block_sum<WARPS>(sum, buf[0]) / dim;
    float sq = 0.f;
#pragma unroll
    for (int k = 0; k < VPT; k++) {
        const int first = (t + k * NT) * VEC - lead;
#pragma unroll
        for (int i = 0; i < VEC; i++) {
            v[k][i] -= mean;
            if (first + i >= 0 && first + i < dim) sq += v[k][i] * v[k][i];
        }
    }
    const float var = block_sum<WARPS>(sq, buf[1]) / dim;
    const float rstd = 1.f / sqrtf(var + eps);
    if (t == 0) {
        if (mean_out) mean_out[r] = mean;
        if (rstd_out) rstd_out[r] = rstd;
    }
    const bool same = row_lead(yr) == lead;
#pragma unroll
    for (int k = 0; k < VPT; k++) {
        const int first = (t + k * NT) * VEC - lead;
        if (first >= dim) continue;
        float o[VEC];
#pragma unroll
        for (int i = 0; i < VEC; i++) {
            const int c = first + i;
            const bool in = c >= 0 && c < dim;
            o[i] = v[k][i] * rstd * (gamma && in ? __ldg(gamma + c) : 1.f) + (beta && in ? __ldg(beta + c) : 0.f);
        }
        if (same) {
            store_block(yr, first, dim, Elem<T>::pack(o));
        } else {
#pragma unroll
            for (int i = 0; i < VEC; i++)
                if (first + i >= 0 && first + i < dim) yr[first + i] = Elem<T>::from(o[i]);
        }
    }
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
    const float mean = block_sum<32>(sum, buf[0]) / dim;
    float sq = 0.f;
    for (int c = threadIdx.x; c < dim; c += 1024) {
        const float d = Elem<T>::to(xr[c]) - mean;
        sq += d * d;
    }
    const float rstd = 1.f / sqrtf(block_sum<32>(sq, buf[1]) / dim + eps);
    if (threadIdx.x == 0) {
        if (mean_out) mean_out[r] = mean;
        if (rstd_out) rstd_out[r] = rstd;
    }
    for (int c = threadIdx.x; c < dim; c += 1024)
        yr[c] = Elem<T>::from((Elem<T>::to(xr[c]) - mean) * rstd * (gamma ? gamma[c] : 1.f) + (beta ? beta[c] : 0.f));
}

constexpr int kNormElems = 16;     // columns per thread of the fused backward kernel
constexpr int kNormMaxThreads = 512;
constexpr int kNormSms = 148;      // the workspace holds one pair of sums per CTA of a grid over this many SMs

// One CTA per residue of rows and slot; period: rows after which the start addresses repeat modulo 16 bytes.
template <typename T, int NT>
__global__ void __launch_bounds__(NT)
layernorm_backward_kernel(const T* dy, const T* x, const float* __restrict__ mean, const float* __restrict__ rstd,
                          const float* __restrict__ gamma, T* dx, float* __restrict__ partial, int64_t rows, int dim,
                          int64_t ld_x, int64_t ld_dy, int64_t ld_dx, int period, int add_dx) {
    constexpr int VEC = Elem<T>::VEC, VPT = kNormElems / VEC, WARPS = NT / 32;
    __shared__ float buf[2][2][WARPS];
    const int t = threadIdx.x;
    const int residue = blockIdx.x % period;
    const int lead = row_lead(x + residue * ld_x);
    float dg[VPT][VEC], db[VPT][VEC], ga[VPT][VEC];
#pragma unroll
    for (int k = 0; k < VPT; k++) {
        const int first = (t + k * NT) * VEC - lead;
#pragma unroll
        for (int i = 0; i < VEC; i++) {
            const int c = first + i;
            dg[k][i] = db[k][i] = 0.f;
            ga[k][i] = c >= 0 && c < dim ? (gamma ? gamma[c] : 1.f) : 0.f;
        }
    }
    int turn = 0;
    const int64_t step = static_cast<int64_t>(gridDim.x / period) * period;
    for (int64_t r = blockIdx.x; r < rows; r += step, turn ^= 1) {
        const T* xr = x + r * ld_x;
        const T* dyr = dy + r * ld_dy;
        const float mu = mean[r], rs = rstd[r];
        uint4 ux[VPT], ud[VPT];
#pragma unroll
        for (int k = 0; k < VPT; k++) {
            const int first = (t + k * NT) * VEC - lead;
            ux[k] = ud[k] = make_uint4(0, 0, 0, 0);
            if (first < dim) {
                ux[k] = load_block(xr, first, dim);
                ud[k] = load_block(dyr, first, dim);
            }
        }
        float sg = 0.f, sgh = 0.f;
#pragma unroll
        for (int k = 0; k < VPT; k++) {
            float fx[VEC], fd[VEC];
            Elem<T>::unpack(ux[k], fx);
            Elem<T>::unpack(ud[k], fd);
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                const float h = (fx[i] - mu) * rs, g = fd[i] * ga[k][i];
                sg += g;
                sgh += g * h;
                dg[k][i] += fd[i] * h;
                db[k][i] += fd[i];
            }
        }
        if (!dx) continue;
        sg = warp_sum(sg);
        sgh = warp_sum(sgh);
        if (WARPS > 1) {
            if ((t & 31) == 0) {
                buf[turn][0][t >> 5] = sg;
                buf[turn][1][t >> 5] = sgh;
            }
            __syncthreads();
            sg = sgh = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; w++) {
                sg += buf[turn][0][w];
                sgh += buf[turn][1][w];
            }
        }
        sg /= dim;
        sgh /= dim;
        T* dxr = dx + r * ld_dx;
#pragma unroll
        for (int k = 0; k < VPT; k++) {
            const int first = (t + k * NT) * VEC - lead;
            if (first >= dim) continue;
            float fx[VEC], fd[VEC];
            Elem<T>::unpack(ux[k], fx);
            Elem<T>::unpack(ud[k], fd);
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                const float h = (fx[i] - mu) * rs;
                fd[i] = rs * (fd[i] * ga[k][i] - sg - h * sgh);
            }
            if (add_dx) {
                Elem<T>::unpack(load_block(dxr, first, dim), fx);
#pragma unroll
                for (int i = 0; i < VEC; i++) fd[i] += fx[i];
            }
            store_block(dxr, first, dim, Elem<T>::pack(fd));
        }
    }
    if (!partial) return;
    float* pg = partial + static_cast<int64_t>(blockIdx.x) * 2 * dim;
#pragma unroll
    for (int k = 0; k < VPT; k++) {
        const int first = (t + k * NT) * VEC - lead;
#pragma unroll
        for (int i = 0; i < VEC; i++) {
            const int c = first + i;
            if (c >= 0 && c < dim) {
                pg[c] = dg[k][i];
                pg[dim + c] = db[k][i];
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
    __shared__ float buf[2][16];
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
    sg = block_sum<16>(sg, buf[0]) / dim;
    sgh = block_sum<16>(sgh, buf[1]) / dim;
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
#pragma unroll 4
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

// CTAs of the fused backward kernel for this row length, threads per CTA; 0 threads: the row is too long.
static int norm_threads(int64_t dim, int vec) {
    const int64_t need = (dim + vec - 1 + kNormElems - 1) / kNormElems;  // the first block may be partly before the row
    for (int nt = 32; nt <= kNormMaxThreads; nt *= 2)
        if (need <= nt) return nt;
    return 0;
}
static int64_t norm_parts(const nzb_layernorm_desc* d) {
    const int nt = norm_threads(d->dim, d->dtype == NZB_F32 ? 4 : 8);
    if (nt == 0) return d->rows < 64 ? d->rows : 64;
    int64_t ctas = (int64_t)kNormSms * (1024 / nt);
    if (ctas > d->rows) ctas = d->rows;
    return ctas < 8 ? 8 : ctas;  // at least one per residue
}

template <typename T, int NT, int VPT>
static void launch_norm(const nzb_layernorm_desc* d, const void* x, const float* gamma, const float* beta, void* y,
                        float* mean, float* rstd, cudaStream_t s) {
    const unsigned blocks = (unsigned)(NT == 32 ? (d->rows + 7) / 8 : d->rows);
    layernorm_kernel<T, NT, VPT><<<blocks, NT == 32 ? 256 : NT, 0, s>>>(static_cast<const T*>(x), gamma, beta, static_cast<T*>(y),
                                                                        mean, rstd, d->rows, (int)d->dim, d->ld_x, d->ld_y, d->eps);
}

template <typename T, int NT>
static void launch_norm_backward(const nzb_layernorm_desc* d, const void* dy, const void* x, const float* mean,
                                 const float* rstd, const float* gamma, void* dx, float* partial, int period, unsigned ctas,
                                 cudaStream_t s) {
    layernorm_backward_kernel<T, NT><<<ctas, NT, 0, s>>>(static_cast<const T*>(dy), static_cast<const T*>(x), mean, rstd, gamma,
                                                         static_cast<T*>(dx), partial, d->rows, (int)d->dim, d->ld_x, d->ld_y,
                                                         d->ld_dx, period, !d->overwrite_dx);
}

}  // namespace nzb

using namespace nzb;

extern "C" {

int nzb_layernorm_forward(const nzb_layernorm_desc* d, const void* x, const float* gamma, const float* beta, void* y,
                          float* mean, float* rstd, void* stream) {
    int rc = check_layernorm(d);
    if (rc != NZB_OK) return rc;
    if (d->rows == 0 || d->dim == 0) return NZB_OK;
    if (!x || !y) return fail(NZB_ERR_BAD_ARG, "x and y must be non-null");
    const int64_t size = dtype_size(d->dtype);
    if (!aligned_to(x, size) || !aligned_to(y, size)) return fail(NZB_ERR_BAD_ARG, "pointer is not a multiple of its element's size");
    DeviceState* ds;
    rc = get_device_state(&ds);
    if (rc != NZB_OK) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    NZB_DISPATCH_DTYPE(d->dtype, T, {
        constexpr int VEC = Elem<T>::VEC;
        const bool aligned = aligned_to(x, 16) && d->ld_x * size % 16 == 0;
        const int64_t n = (d->dim + (aligned ? 0 : VEC - 1) + VEC - 1) / VEC;  // 16-byte blocks of a row
        if (n <= 32) launch_norm<T, 32, 1>(d, x, gamma, beta, y, mean, rstd, s);
        else if (n <= 64) launch_norm<T, 32, 2>(d, x, gamma, beta, y, mean, rstd, s);
        else if (n <= 128) launch_norm<T, 32, 4>(d, x, gamma, beta, y, mean, rstd, s);
        else if (n <= 256) launch_norm<T, 128, 2>(d, x, gamma, beta, y, mean, rstd, s);
        else if (n <= 512) launch_norm<T, 128, 4>(d, x, gamma, beta, y, mean, rstd, s);
        else if (n <= 1024) launch_norm<T, 256, 4>(d, x, gamma, beta, y, mean, rstd, s);
        else if (n <= 2048) launch_norm<T, 512, 4>(d, x, gamma, beta, y, mean, rstd, s);
        else if (n <= 4096) launch_norm<T, 1024, 4>(d, x, gamma, beta, y, mean, rstd, s);
        else layernorm_long_kernel<T><<<(unsigned)d->rows, 1024, 0, s>>>(static_cast<const T*>(x), gamma, beta, static_cast<T*>(y), mean, rstd, (int)d->dim, d->ld_x, d->ld_y, d->eps);
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
    const int nt = together ? norm_threads(d->dim, d->dtype == NZB_F32 ? 4 : 8) : 0;
    if (nt) {
        const int period = d->ld_x * size % 16 == 0 ? 1 : (int)(16 / size);
        parts = parts / period * period;  // whole rounds of the residues: norm_parts gives eight at least
        NZB_DISPATCH_DTYPE(d->dtype, T, {
            if (nt == 32) launch_norm_backward<T, 32>(d, dy, x, mean, rstd, gamma, dx, partial, period, (unsigned)parts, s);
            else if (nt == 64) launch_norm_backward<T, 64>(d, dy, x, mean, rstd, gamma, dx, partial, period, (unsigned)parts, s);
            else if (nt == 128) launch_norm_backward<T, 128>(d, dy, x, mean, rstd, gamma, dx, partial, period, (unsigned)parts, s);
            else if (nt == 256) launch_norm_backward<T, 256>(d, dy, x, mean, rstd, gamma, dx, partial, period, (unsigned)parts, s);
            else launch_norm_backward<T, 512>(d, dy, x, mean, rstd, gamma, dx, partial, period, (unsigned)parts, s);
        });
    } else {
        NZB_DISPATCH_DTYPE(d->dtype, T, {
            const T* xp = static_cast<const T*>(x);
            const T* dyp = static_cast<const T*>(dy);
            if (params) {
                if (parts > 64) parts = 64;
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
