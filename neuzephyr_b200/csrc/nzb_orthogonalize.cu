// Orthogonalised update of a weight matrix by Newton-Schulz products, and the Muon step that applies it. Beside
// the Adam and SGD steps.
//
//   X = G / (|G|_F + eps); steps times: A = X X^T, B = c1 A + c2 A A, X = c0 X + B X      (rows <= cols)
// and A = X^T X, X = c0 X + X B for a tall matrix: either operand of a product may be K-major or MN-major, so no
// pass transposes anything. S is the short side, L the long one; a step costs 2 S^2 L + 2 S^3 + 2 S^2 L operations,
// of which the symmetric A and B need one half each.
//
// Precision. The recurrence multiplies small singular values by c0 (3.4) a step, and with them whatever noise the
// roundings put there: 140 times what the first step rounds off, in the directions that a matrix of low rank leaves empty. So
// X is held in fp32, X = (c0 + B_ii) X32 + (B - diag B) X, and the products' operands as pairs of fp16 numbers, high =
// fp16(v) and low = fp16(v - high), 22 bits together, of which a product takes high high + high low + low high. X and A
// are stored times 2^12, so that entries down to 2^-26 keep 11 bits in each part, B as it is (its pairs leave out less than
// 2^-25, where c0 X outweighs it by far); B's diagonal, which carries most of B once X is near orthogonal, multiplies the
// fp32 X. Against 64 bits (Frobenius norm): 1e-5 at 256 x 512, 2e-5 at 1000 x 1400, 6e-5 at 4096 x 4096 (the tensor cores'
// sums are what is left), and for matrices of rank one, where fp32 products do little better, 1e-4, 3e-4 and 9e-4. The
// high parts alone take 0.4 of the time at large sides and are 5e-4 to 1e-3 off, but up to 4e-2 for matrices of rank one
// (5 x 144; with uneven entries 2331 x 2103 too).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "nzb_elem.cuh"
#include "nzb_gemm_tile.cuh"
#include "nzb_internal.h"
#include "nzb_ptx.cuh"

namespace nzb {

constexpr float kNsScale = 4096.f;            // 2^12: what X (all copies) and A are multiplied by
constexpr float kNsUnscale = 1.f / 4096.f;

enum { NS_GRAM = 0, NS_POLY = 1, NS_APPLY = 2 };
enum { NS_OUT_STATE = 0, NS_OUT_F32 = 1, NS_OUT_F16 = 2, NS_OUT_BF16 = 3, NS_OUT_WEIGHT = 4 };

struct NsParams {
    int32_t M, N;              // output extents
    int32_t k_blocks, last_ksteps;
    int32_t tiles_m, tiles_n, group_m;
    int32_t a_mn, b_mn;
    int32_t symmetric;         // A and B by their lower triangle of (square) tiles, mirrored; 0: every tile
    int32_t by_column;         // NS_APPLY of a tall matrix: the diagonal belongs to the columns
    int32_t out_kind, out_vec; // NS_APPLY
    int64_t tiles, tiles_per_matrix;
    int32_t splits;            // NS_GRAM: CTAs that share a tile, each with a stretch of the contraction (sums in `partial`)
    float* partial;            // [split][matrix][rows and columns of the short side in blocks of 32 x 32]
    int64_t stride_part, batch;
    float c0, c1, c2;
    __half* out16;             // 2^12 A, B or the next 2^12 X: first all matrices' high parts, then their low parts
    int64_t ld16, stride16, low16;  // low16: from a high part to its low part
    const __half* gram;        // NS_POLY: A times 2^12, same layout as out16
    float* diag;               // c0 + B_ii, `short_side` per matrix
    int64_t short_side;
    float* X32;
    int64_t ldx, stridex;
    void* out;                 // NS_APPLY, last step
    int64_t ld_out, stride_out;
    float w_keep, w_step;      // NS_OUT_WEIGHT: w = w_keep w - w_step x
    int* status;
};

// A tile is BM x BN per CTA (PAIR: two CTAs share one of twice the rows).
template <bool PAIR_, int BN_>
struct NsCfg {
    static constexpr bool PAIR = PAIR_;
    static constexpr int BM = PAIR ? 256 : 128, BN = BN_;
    static constexpr int STAGES = BN >= 128 ? 3 : 4;
    // two or four per quarter of the tensor-memory lanes. The epilogue is a long chain per warp (tensor memory, shared
    // memory, memory): on a 256-wide tile, with one part to write, eight warps took 15000 cycles, whatever they left out,
    // sixteen 7500
    static constexpr int EPI_WARPS = BN >= 128 ? 16 : 8;
    static constexpr int COLS = BN * 4 / EPI_WARPS;   // columns of a warp
    static constexpr int THREADS = 64 + 32 * EPI_WARPS;
    static constexpr int B_ROWS = PAIR ? BN / 2 : BN; // rows of B that a CTA loads
    static constexpr int A_BYTES = 128 * 64 * 2;      // per k block of 64 and part
    static constexpr int B_BYTES = B_ROWS * 64 * 2;
    static constexpr int STAGE_BYTES = 2 * (A_BYTES + B_BYTES);  // A high, A low, B high, B low
    static constexpr int EPI_BYTES = EPI_WARPS * 2048;  // 32 x 32 fp16 entries per warp
    static constexpr int SMEM_BYTES = 1024 + STAGES * STAGE_BYTES + EPI_BYTES + 256;
    static constexpr int TMEM_COLS = 2 * BN;
    static_assert(BN >= 64, "an MN-major operand is loaded in boxes of 64 columns");
    static_assert(SMEM_BYTES <= 232448, "exceeds the 227 KB shared memory of an sm_100 CTA");
};

// The tile of a work item and the k blocks [k0, k1) it covers.
template <int MODE>
__device__ __forceinline__ int64_t ns_tile(const NsParams& p, int64_t item, int32_t& k0, int32_t& k1) {
    k0 = 0;
    k1 = p.k_blocks;
    if (MODE != NS_GRAM || p.splits == 1) return item;
    const int32_t split = static_cast<int32_t>(item % p.splits);
    k0 = static_cast<int32_t>(static_cast<int64_t>(p.k_blocks) * split / p.splits);
    k1 = static_cast<int32_t>(static_cast<int64_t>(p.k_blocks) * (split + 1) / p.splits);
    return item / p.splits;
}

// Symmetric outputs: tile numbers run over the lower triangle, row of tiles by row of tiles.
template <int MODE>
__device__ __forceinline__ void ns_decode(const NsParams& p, int64_t tile, int32_t& mt, int32_t& nt, int32_t& b) {
    b = static_cast<int32_t>(tile / p.tiles_per_matrix);
    const int32_t rem = static_cast<int32_t>(tile - b * p.tiles_per_matrix);
    if (MODE == NS_APPLY || !p.symmetric) {
        const int32_t group = p.group_m * p.tiles_n, g = rem / group, first = g * p.group_m;
        const int32_t gm = min(p.tiles_m - first, p.group_m), within = rem - g * group;
        mt = first + within % gm;
        nt = within / gm;
    } else {
        int32_t m = static_cast<int32_t>((sqrtf(8.f * rem + 1.f) - 1.f) * 0.5f);
        while (m * (m + 1) / 2 > rem) m--;
        while ((m + 1) * (m + 2) / 2 <= rem) m++;
        mt = m;
        nt = rem - m * (m + 1) / 2;
    }
}

// 32 x 32 fp16 entries in shared memory, 64 bytes a row: 16-byte piece j of row r lies at j ^ (r / 2 & 3), so that a lane per
// row and four lanes per row both go without bank conflicts.
__device__ __forceinline__ uint4* ns_piece(float* stage, int r, int j) { return reinterpret_cast<uint4*>(stage) + r * 4 + (j ^ (r >> 1 & 3)); }

// Writes 32 x 32 entries of one part, a row per lane in h, at (row0, col0) of an A or B and, with `mirror`, their mirror image. Rows
// go to memory four lanes to 64 bytes, by way of shared memory (a lane per row touches 32 lines an instruction: 19000
// cycles for a 256 x 256 tile of B).
__device__ __forceinline__ void ns_store_block(const NsParams& p, __half* out, float* stage, int lane, int32_t row0, int32_t col0,
                                               const __half2 (&h)[16], bool mirror) {
    const int pr = lane >> 2, pj = lane & 3;  // this lane's row (of eight) and piece
    // Rows r0 .. r0 + 31 (below `rows`) of the entries in shared memory, to columns c0 .. of the matrix.
    const auto put = [&](int32_t r0, int32_t rows, int32_t c0) {
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint4 u = *ns_piece(stage, 8 * i + pr, pj);
            if (r0 + 8 * i + pr < rows && c0 + 8 * pj < p.ld16) *reinterpret_cast<uint4*>(out + static_cast<int64_t>(r0 + 8 * i + pr) * p.ld16 + c0 + 8 * pj) = u;
        }
        __syncwarp();
    };
    const uint4* own = reinterpret_cast<const uint4*>(h);
#pragma unroll
    for (int j = 0; j < 4; j++) *ns_piece(stage, lane, j) = own[j];
    put(row0, p.M, col0);
    if (!mirror) return;
    // entry (row, col) to (col, row). Two lanes trade halves so that each holds a pair of rows: the even lane of column 2j,
    // the odd one of column 2j + 1; a column's 32 rows become a row of 64 bytes.
#pragma unroll
    for (int j = 0; j < 16; j++) {
        const __half give = lane & 1 ? __low2half(h[j]) : __high2half(h[j]);
        const __half got = __ushort_as_half(__shfl_xor_sync(0xffffffffu, __half_as_ushort(give), 1));
        const __half2 two = lane & 1 ? __halves2half2(got, __high2half(h[j])) : __halves2half2(__low2half(h[j]), got);
        reinterpret_cast<__half2*>(ns_piece(stage, 2 * j + (lane & 1), lane >> 3))[lane >> 1 & 3] = two;
    }
    put(col0, p.N, row0);
}

// A pair of numbers as fp16 high parts and what they leave, in fp16 too.
__device__ __forceinline__ __half2 ns_low(float x, float y, __half2 high) {
    const float2 f = __half22float2(high);
    return __floats2half2_rn(x - f.x, y - f.y);
}

// X32 (2^12 X) in the order the epilogue holds it: blocks of 32 x 32, in each the rows' first four columns, then the rows' next
// four, so that a lane per row reads and writes 512 contiguous bytes an instruction. Offset of row r's columns c .. c + 3.
__host__ __device__ __forceinline__ int64_t ns_state_at(int64_t r, int64_t c, int64_t ldx) {
    return ((r >> 5) * (ldx >> 5) + (c >> 5)) * 1024 + (c >> 2 & 7) * 128 + (r & 31) * 4;
}

// Drains 32 rows x a warp's columns of a finished A or B tile: every lane holds one row, 32 columns at a time. `ready` waits for
// the accumulator; what else a group of columns needs is loaded before that.
template <class Cfg, int MODE, class Ready>
__device__ __forceinline__ bool ns_drain_symmetric(const NsParams& p, uint32_t tmem, float* stage, int lane, int32_t b, int32_t row0,
                                                   int32_t col_first, bool mirror, int32_t split, int64_t batch, Ready ready) {
    using namespace ptx;
    __half* out = p.out16 + b * p.stride16;
    const int32_t row = row0 + lane;
    const int pr = lane >> 2, pj = lane & 3;
    const __half* gram = p.gram + b * p.stride16;
    uint4 g[2][4];  // A's high and low parts
    const auto fetch = [&](int32_t col0) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int32_t r = row0 + 8 * i + pr;
            const __half* from = gram + static_cast<int64_t>(r) * p.ld16 + col0 + 8 * pj;
            const bool in = r < p.M && col0 < p.N;
            g[0][i] = in ? *reinterpret_cast<const uint4*>(from) : make_uint4(0, 0, 0, 0);
            g[1][i] = in ? *reinterpret_cast<const uint4*>(from + p.low16) : make_uint4(0, 0, 0, 0);
        }
    };
    const float k1 = p.c1 * kNsUnscale, k2 = p.c2 * kNsUnscale * kNsUnscale;
    if (MODE == NS_POLY) fetch(col_first);
    if (!ready()) return false;
#pragma unroll 1
    for (int c0 = 0; c0 < Cfg::COLS; c0 += 32) {
        const int32_t col0 = col_first + c0;
        if (col0 >= p.N) break;  // warp-uniform; the padded leading dimension covers a started group of 32
        uint32_t v[32];
        tmem_ld_32x32(tmem + c0, v);
        tmem_ld_wait();
        if (MODE == NS_GRAM && p.splits > 1) {
            // a part of the sum, as the accumulator has it
            if (row0 < p.M) {
                float4* to = reinterpret_cast<float4*>(p.partial + (split * batch + b) * p.stride_part + ns_state_at(row, col0, p.ld16));
#pragma unroll
                for (int j = 0; j < 8; j++)
                    to[j * 32] = make_float4(__uint_as_float(v[4 * j]), __uint_as_float(v[4 * j + 1]), __uint_as_float(v[4 * j + 2]), __uint_as_float(v[4 * j + 3]));
            }
            continue;
        }
        float x[32];
        if (MODE == NS_GRAM) {
#pragma unroll
            for (int j = 0; j < 32; j++) x[j] = __uint_as_float(v[j]) * kNsUnscale;
        } else {
#pragma unroll
            for (int j = 0; j < 32; j++) x[j] = k2 * __uint_as_float(v[j]);
#pragma unroll
            for (int part = 0; part < 2; part++) {
#pragma unroll
                for (int i = 0; i < 4; i++) *ns_piece(stage, 8 * i + pr, pj) = g[part][i];
                __syncwarp();
                uint4 mine[4];
#pragma unroll
                for (int j = 0; j < 4; j++) mine[j] = *ns_piece(stage, lane, j);
                __syncwarp();
                const __half2* gh = reinterpret_cast<const __half2*>(mine);
#pragma unroll
                for (int j = 0; j < 16; j++) {
                    const float2 a = __half22float2(gh[j]);
                    x[2 * j] = fmaf(k1, a.x, x[2 * j]);
                    x[2 * j + 1] = fmaf(k1, a.y, x[2 * j + 1]);
                }
            }
#pragma unroll
            for (int j = 0; j < 32; j++) {
                if (row != col0 + j) continue;
                if (row < p.M) p.diag[b * p.short_side + row] = p.c0 + x[j];
                x[j] = 0.f;
            }
        }
        __half2 h[16];
#pragma unroll
        for (int j = 0; j < 16; j++) h[j] = __floats2half2_rn(x[2 * j], x[2 * j + 1]);
        ns_store_block(p, out, stage, lane, row0, col0, h, mirror);
#pragma unroll
        for (int j = 0; j < 16; j++) h[j] = ns_low(x[2 * j], x[2 * j + 1], h[j]);
        ns_store_block(p, out + p.low16, stage, lane, row0, col0, h, mirror);
        if (MODE == NS_POLY && c0 + 32 < Cfg::COLS) fetch(col0 + 32);
    }
    return true;
}

// Drains 32 rows x a warp's columns of a finished B X tile and completes the step, x = diag * x + product, or writes the
// result's elements. X32 does not depend on the product, so a group's part is on its way before the accumulator is
// ready, the next group's before this one is written. Shared memory, which the products keep busy, only turns the fp16
// rows around.
template <class Cfg, class Ready>
__device__ __forceinline__ bool ns_drain_apply(const NsParams& p, uint32_t tmem, float* stage, int lane, int32_t b,
                                               int32_t row0, int32_t col_first, Ready ready) {
    using namespace ptx;
    const float* diag = p.diag + b * p.short_side;
    const int32_t row = row0 + lane;
    const bool row_ok = row < p.M;
    float* X = p.X32 + b * p.stridex;
    const int pr = lane >> 2, pj = lane & 3;
    float4 old[8];
    float dcol = 0.f;  // by column: this lane's of the group
    const auto fetch = [&](int32_t col0) {
        if (p.by_column) dcol = col0 + lane < p.N ? diag[col0 + lane] : 0.f;
        if (!row_ok || col0 >= p.N) return;
        const float4* from = reinterpret_cast<const float4*>(X + ns_state_at(row, col0, p.ldx));
#pragma unroll
        for (int j = 0; j < 8; j++) old[j] = from[j * 32];
    };
    fetch(col_first);
    const float dr = !p.by_column && row_ok ? diag[row] : 0.f;
    if (!ready()) return false;
#pragma unroll 1
    for (int c0 = 0; c0 < Cfg::COLS; c0 += 32) {
        const int32_t col0 = col_first + c0;
        if (col0 >= p.N) break;  // warp-uniform
        if (p.by_column) {
            stage[lane] = dcol;
            __syncwarp();
        }
        uint32_t v[32];
        tmem_ld_32x32(tmem + c0, v);
        tmem_ld_wait();
        float4 x[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float4 d = p.by_column ? reinterpret_cast<const float4*>(stage)[j] : make_float4(dr, dr, dr, dr);
            x[j].x = fmaf(d.x, old[j].x, __uint_as_float(v[4 * j]));
            x[j].y = fmaf(d.y, old[j].y, __uint_as_float(v[4 * j + 1]));
            x[j].z = fmaf(d.z, old[j].z, __uint_as_float(v[4 * j + 2]));
            x[j].w = fmaf(d.w, old[j].w, __uint_as_float(v[4 * j + 3]));
        }
        if (p.by_column) __syncwarp();
        if (c0 + 32 < Cfg::COLS) fetch(col0 + 32);
        if (p.out_kind == NS_OUT_STATE) {
            if (row_ok) {
                float4* to = reinterpret_cast<float4*>(X + ns_state_at(row, col0, p.ldx));
#pragma unroll
                for (int j = 0; j < 8; j++) to[j * 32] = x[j];
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                x[j].x *= kNsUnscale; x[j].y *= kNsUnscale; x[j].z *= kNsUnscale; x[j].w *= kNsUnscale;
            }
        }
        if (p.out_kind == NS_OUT_F32 || p.out_kind == NS_OUT_WEIGHT) {
            // once per pass, so a lane writes its row's 128 bytes itself
            float* to = static_cast<float*>(p.out) + b * p.stride_out + static_cast<int64_t>(row) * p.ld_out + col0;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                float f[4] = {x[j].x, x[j].y, x[j].z, x[j].w};
                if (!row_ok) continue;
                if (p.out_vec && col0 + 4 * j + 4 <= p.N) {
                    float4* at = reinterpret_cast<float4*>(to) + j;
                    if (p.out_kind == NS_OUT_WEIGHT) {
                        const float4 w = *at;
                        *at = make_float4(fmaf(-p.w_step, f[0], p.w_keep * w.x), fmaf(-p.w_step, f[1], p.w_keep * w.y),
                                          fmaf(-p.w_step, f[2], p.w_keep * w.z), fmaf(-p.w_step, f[3], p.w_keep * w.w));
                    } else {
                        *at = x[j];
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (col0 + 4 * j + i < p.N) to[4 * j + i] = p.out_kind == NS_OUT_WEIGHT ? fmaf(-p.w_step, f[i], p.w_keep * to[4 * j + i]) : f[i];
                }
            }
            continue;
        }
        const bool state = p.out_kind == NS_OUT_STATE;
        const int64_t ld = state ? p.ld16 : p.ld_out;
        uint16_t* out = (state ? reinterpret_cast<uint16_t*>(p.out16) + b * p.stride16 : static_cast<uint16_t*>(p.out) + b * p.stride_out) +
                        static_cast<int64_t>(row0 + pr) * ld + col0 + 8 * pj;
        const bool vec = state || (p.out_vec && col0 + 8 * pj + 8 <= p.N);  // the state's padded rows hold whole groups
        __half2 h[16];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            if (p.out_kind == NS_OUT_BF16) {
                const __nv_bfloat162 lo = __floats2bfloat162_rn(x[j].x, x[j].y), hi = __floats2bfloat162_rn(x[j].z, x[j].w);
                h[2 * j] = *reinterpret_cast<const __half2*>(&lo);
                h[2 * j + 1] = *reinterpret_cast<const __half2*>(&hi);
            } else {
                h[2 * j] = __floats2half2_rn(x[j].x, x[j].y);
                h[2 * j + 1] = __floats2half2_rn(x[j].z, x[j].w);
            }
        }
        // a result's rows, or the state's high parts and then its low parts
#pragma unroll 1
        for (int part = 0; part < (state ? 2 : 1); part++, out += p.low16) {
            if (part) {
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    h[2 * j] = ns_low(x[j].x, x[j].y, h[2 * j]);
                    h[2 * j + 1] = ns_low(x[j].z, x[j].w, h[2 * j + 1]);
                }
            }
            const uint4* own = reinterpret_cast<const uint4*>(h);
#pragma unroll
            for (int j = 0; j < 4; j++) *ns_piece(stage, lane, j) = own[j];
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint4 u = *ns_piece(stage, 8 * i + pr, pj);
                if (row0 + 8 * i + pr >= p.M) continue;
                if (vec) {
                    *reinterpret_cast<uint4*>(out + 8 * i * ld) = u;
                } else {
                    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                    for (int k = 0; k < 8; k++)
                        if (col0 + 8 * pj + k < p.N) out[8 * i * ld + k] = static_cast<uint16_t>(w[k / 2] >> (16 * (k & 1)));
                }
            }
            __syncwarp();
        }
    }
    return true;
}

// One product of all matrices. CTA layout (persistent over the tiles): warp 0 TMA producer, warp 1 tensor-memory
// allocator and MMA issuer, the others epilogue; two accumulators, so that a tile's epilogue runs
// under the next tile's products. PAIR: two CTAs share a 256 x 256 tile (each loads its 128 rows of both operands).
// Every wait is bounded; on expiry the CTA raises its abort flag, waits for its copies in flight, frees its tensor
// memory and returns with NZB_ERR_DEVICE_TIMEOUT in the status word.
template <class Cfg, int MODE>
__global__ void __launch_bounds__(Cfg::THREADS, 1)
ns_product_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const NsParams p) {
    using namespace ptx;
    constexpr bool PAIR = Cfg::PAIR;
    constexpr int STAGES = Cfg::STAGES;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    float* epi = reinterpret_cast<float*>(smem + STAGES * Cfg::STAGE_BYTES);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + STAGES * Cfg::STAGE_BYTES + Cfg::EPI_BYTES);
    uint64_t* full = bars;
    uint64_t* empty = bars + STAGES;
    uint64_t* tfull = bars + 2 * STAGES;
    uint64_t* tempty = bars + 2 * STAGES + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * STAGES + 4);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = PAIR ? cluster_ctarank() : 0;
    const int64_t first_tile = PAIR ? blockIdx.x >> 1 : blockIdx.x, step = PAIR ? gridDim.x >> 1 : gridDim.x;

    if (threadIdx.x == 0) {
        prefetch_tensormap(&tmA);
        prefetch_tensormap(&tmB);
        for (int s = 0; s < STAGES; s++) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int a = 0; a < 2; a++) {
            mbar_init(&tfull[a], 1);
            mbar_init(&tempty[a], (PAIR ? 2 : 1) * Cfg::EPI_WARPS);
        }
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        if constexpr (PAIR) {
            tmem_alloc_pair(tmem_slot, Cfg::TMEM_COLS);
            tmem_relinquish_pair();
        } else {
            tmem_alloc(tmem_slot, Cfg::TMEM_COLS);
            tmem_relinquish();
        }
    }
    tc_fence_before();
    if constexpr (PAIR) cluster_sync_all();
    else __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    // everything above ran under the previous kernel's end; its results are there from here on
    kernel_wait_previous();
    kernel_allow_next();

    if (warp == 0) {
        uint32_t it = 0;
        bool ok = true;
        for (int64_t item = first_tile; item < p.tiles * p.splits && ok; item += step) {
            int32_t mt, nt, b, k0, k1;
            ns_decode<MODE>(p, ns_tile<MODE>(p, item, k0, k1), mt, nt, b);
            const int32_t row_a = mt * Cfg::BM + (int32_t)rank * 128, row_b = nt * Cfg::BN + (int32_t)rank * Cfg::B_ROWS;
            for (int32_t kb = k0; kb < k1; kb++, it++) {
                const uint32_t s = it % STAGES, ph = (it / STAGES) & 1;
                if (!mbar_wait_warp(&empty[s], ph ^ 1, abort_flag)) {
                    ok = false;
                    break;
                }
                if (elect_one()) {
                    uint8_t* sa = smem + s * Cfg::STAGE_BYTES;
                    uint8_t* sb = sa + 2 * Cfg::A_BYTES;
                    const int32_t low = b + static_cast<int32_t>(p.batch);  // the low parts follow all high parts
                    if constexpr (PAIR) {
                        const uint32_t leader_full = map_to_cta(smem_u32(&full[s]), 0);
                        if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * Cfg::STAGE_BYTES);
                        load_operand_pair<128>(sa, &tmA, p.a_mn, kb * 64, row_a, b, leader_full);
                        load_operand_pair<Cfg::B_ROWS>(sb, &tmB, p.b_mn, kb * 64, row_b, b, leader_full);
                        load_operand_pair<128>(sa + Cfg::A_BYTES, &tmA, p.a_mn, kb * 64, row_a, low, leader_full);
                        load_operand_pair<Cfg::B_ROWS>(sb + Cfg::B_BYTES, &tmB, p.b_mn, kb * 64, row_b, low, leader_full);
                    } else {
                        mbar_arrive_expect_tx(&full[s], Cfg::STAGE_BYTES);
                        load_operand<128>(sa, &tmA, p.a_mn, kb * 64, row_a, b, &full[s]);
                        load_operand<Cfg::B_ROWS>(sb, &tmB, p.b_mn, kb * 64, row_b, b, &full[s]);
                        load_operand<128>(sa + Cfg::A_BYTES, &tmA, p.a_mn, kb * 64, row_a, low, &full[s]);
                        load_operand<Cfg::B_ROWS>(sb + Cfg::B_BYTES, &tmB, p.b_mn, kb * 64, row_b, low, &full[s]);
                    }
                }
                __syncwarp();
            }
        }
        if (!ok && rank == 0 && lane == 0) {
            // wait (bounded) for the copies still in flight so none lands after exit
            const uint32_t first = it > (uint32_t)STAGES ? it - STAGES : 0;
            const long long t0 = clock64();
            for (uint32_t j = first; j < it; j++) {
                while (!mbar_try_wait(&full[j % STAGES], (j / STAGES) & 1)) {
                    if (clock64() - t0 > kWaitCycleLimit) break;
                }
            }
        }
    } else if (warp == 1) {
        if (rank == 0) {
            const uint32_t idesc = make_idesc_f16_f32(Cfg::BM, Cfg::BN) | (p.a_mn ? 1u << 15 : 0u) | (p.b_mn ? 1u << 16 : 0u);
            const uint64_t hi_a = desc_high_bits(p.a_mn), hi_b = desc_high_bits(p.b_mn);
            const uint32_t ka = desc_kstep(p.a_mn), kb_step = desc_kstep(p.b_mn);
            uint32_t it = 0, tcount = 0;
            bool ok = true;
            for (int64_t item = first_tile; item < p.tiles * p.splits && ok; item += step, tcount++) {
                int32_t k0, k1;
                ns_tile<MODE>(p, item, k0, k1);
                const uint32_t acc = tcount & 1, aph = (tcount >> 1) & 1;
                if (!mbar_wait_warp(&tempty[acc], aph ^ 1, abort_flag)) break;
                tc_fence_after();
                const uint32_t d_tmem = tmem_base + acc * Cfg::BN;
                for (int32_t kb = k0; kb < k1; kb++, it++) {
                    const uint32_t s = it % STAGES, ph = (it / STAGES) & 1;
                    if (!mbar_wait_warp(&full[s], ph, abort_flag)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t sa = smem_u32(smem + s * Cfg::STAGE_BYTES);
                    const uint64_t da = hi_a | ((sa & 0x3ffff) >> 4);
                    const uint64_t db = hi_b | (((sa + 2 * Cfg::A_BYTES) & 0x3ffff) >> 4);
                    const int32_t ksteps = kb == p.k_blocks - 1 ? p.last_ksteps : 4;
                    if (elect_one()) {
                        // high x high, high x low, low x high; low x low is below fp32's last bit
#pragma unroll
                        for (int term = 0; term < 3; term++) {
                            const uint64_t ta = da + (term == 2 ? Cfg::A_BYTES >> 4 : 0), tb = db + (term == 1 ? Cfg::B_BYTES >> 4 : 0);
                            const uint32_t onto = term || kb > k0 ? 1u : 0u;
                            if constexpr (PAIR) {
                                mma_f16_ss_pair(d_tmem, ta, tb, idesc, onto);
                                if (ksteps > 1) mma_f16_ss_pair(d_tmem, ta + ka, tb + kb_step, idesc, 1u);
                                if (ksteps > 2) mma_f16_ss_pair(d_tmem, ta + 2 * ka, tb + 2 * kb_step, idesc, 1u);
                                if (ksteps > 3) mma_f16_ss_pair(d_tmem, ta + 3 * ka, tb + 3 * kb_step, idesc, 1u);
                            } else {
                                mma_f16_ss(d_tmem, ta, tb, idesc, onto);
                                if (ksteps > 1) mma_f16_ss(d_tmem, ta + ka, tb + kb_step, idesc, 1u);
                                if (ksteps > 2) mma_f16_ss(d_tmem, ta + 2 * ka, tb + 2 * kb_step, idesc, 1u);
                                if (ksteps > 3) mma_f16_ss(d_tmem, ta + 3 * ka, tb + 3 * kb_step, idesc, 1u);
                            }
                        }
                        if constexpr (PAIR) mma_commit_pair(&empty[s]);
                        else mma_commit(&empty[s]);
                    }
                    __syncwarp();
                }
                if (ok && elect_one()) {
                    if constexpr (PAIR) mma_commit_pair(&tfull[acc]);
                    else mma_commit(&tfull[acc]);
                }
                __syncwarp();
            }
        }
    } else {
        const int q = warp & 3;
        float* stage = epi + (warp - 2) * 512;
        uint32_t tcount = 0;
        for (int64_t item = first_tile; item < p.tiles * p.splits; item += step, tcount++) {
            int32_t mt, nt, b, k0, k1;
            ns_decode<MODE>(p, ns_tile<MODE>(p, item, k0, k1), mt, nt, b);
            const uint32_t acc = tcount & 1, aph = (tcount >> 1) & 1;
            const auto ready = [&] {
                if (!mbar_wait_warp(&tfull[acc], aph, abort_flag)) return false;
                tc_fence_after();
                return true;
            };
            const int col_part = ((warp - 2) >> 2) * Cfg::COLS;
            const int32_t row0 = mt * Cfg::BM + (int32_t)rank * 128 + q * 32, col_first = nt * Cfg::BN + col_part;
            const uint32_t tmem = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + acc * Cfg::BN + col_part;
            bool ok;
            if constexpr (MODE == NS_APPLY) ok = ns_drain_apply<Cfg>(p, tmem, stage, lane, b, row0, col_first, ready);
            else ok = ns_drain_symmetric<Cfg, MODE>(p, tmem, stage, lane, b, row0, col_first, p.symmetric && mt != nt, static_cast<int32_t>(item % p.splits), p.batch, ready);
            if (!ok) break;
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if constexpr (PAIR) mbar_arrive_cluster(map_to_cta(smem_u32(&tempty[acc]), 0));
                else mbar_arrive(&tempty[acc]);
            }
        }
    }

    __syncwarp();
    tc_fence_before();
    if constexpr (PAIR) cluster_sync_all();
    else __syncthreads();
    if (threadIdx.x == 0 && *abort_flag) {
        *p.status = NZB_ERR_DEVICE_TIMEOUT;
        __threadfence_system();
    }
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        if constexpr (PAIR) tmem_dealloc_pair(tmem_base, Cfg::TMEM_COLS);
        else tmem_dealloc(tmem_base, Cfg::TMEM_COLS);
    }
}

// Adds the parts of a split A and writes it: a warp per block of 32 x 32 on or below the diagonal, and its mirror image.
__global__ void __launch_bounds__(128)
ns_gram_sum_kernel(const NsParams p) {
    __shared__ float stage[4][512];
    kernel_wait_previous();
    kernel_allow_next();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int32_t side = (p.M + 31) / 32, per_matrix = side * (side + 1) / 2;
    const int64_t block = static_cast<int64_t>(blockIdx.x) * 4 + warp, b = block / per_matrix;
    if (b >= p.batch) return;
    const int32_t rem = static_cast<int32_t>(block - b * per_matrix);
    int32_t m = static_cast<int32_t>((sqrtf(8.f * rem + 1.f) - 1.f) * 0.5f);
    while (m * (m + 1) / 2 > rem) m--;
    while ((m + 1) * (m + 2) / 2 <= rem) m++;
    const int32_t row0 = m * 32, col0 = (rem - m * (m + 1) / 2) * 32;
    const float4* from = reinterpret_cast<const float4*>(p.partial + b * p.stride_part + ns_state_at(row0 + lane, col0, p.ld16));
    float4 sum[8];
#pragma unroll
    for (int j = 0; j < 8; j++) sum[j] = from[j * 32];
#pragma unroll 2
    for (int s = 1; s < p.splits; s++) {
        const float4* part = from + s * (p.batch * p.stride_part / 4);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float4 v = part[j * 32];
            sum[j].x += v.x; sum[j].y += v.y; sum[j].z += v.z; sum[j].w += v.w;
        }
    }
    __half* out = p.out16 + b * p.stride16;
    __half2 h[16];
#pragma unroll
    for (int j = 0; j < 8; j++) {
        sum[j].x *= kNsUnscale; sum[j].y *= kNsUnscale; sum[j].z *= kNsUnscale; sum[j].w *= kNsUnscale;
        h[2 * j] = __floats2half2_rn(sum[j].x, sum[j].y);
        h[2 * j + 1] = __floats2half2_rn(sum[j].z, sum[j].w);
    }
    ns_store_block(p, out, stage[warp], lane, row0, col0, h, row0 != col0);
#pragma unroll
    for (int j = 0; j < 8; j++) {
        h[2 * j] = ns_low(sum[j].x, sum[j].y, h[2 * j]);
        h[2 * j + 1] = ns_low(sum[j].z, sum[j].w, h[2 * j + 1]);
    }
    ns_store_block(p, out + p.low16, stage[warp], lane, row0, col0, h, row0 != col0);
}

// ---- Frobenius norm and first state ---------------------------------------------------------------------------
constexpr int kNormParts = 592;  // partial sums per matrix, at most

// Both elementwise passes go over groups of eight columns. ROWS: neighbouring threads take a row's neighbouring groups
// (reading is all there is); otherwise a CTA takes 32 rows x 64 columns and a warp 8 x 32 of them: 64 bytes and more of
// every row, and whole lines of X32's order.
template <bool ROWS>
struct NsGroups {
    int64_t item, items;
    uint32_t per_row;
    __device__ __forceinline__ NsGroups(int64_t rows, int64_t cols) {
        per_row = static_cast<uint32_t>(ROWS ? (cols + 7) / 8 : (cols + 63) / 64);
        item = ROWS ? static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x : blockIdx.x;
        items = (ROWS ? rows : (rows + 31) / 32) * per_row;
    }
    __device__ __forceinline__ bool more() const { return item < items; }
    __device__ __forceinline__ void next() { item += static_cast<int64_t>(gridDim.x) * (ROWS ? 256 : 1); }
    __device__ __forceinline__ void at(int64_t& r, int64_t& c) const {
        r = items >> 32 ? item / per_row : static_cast<uint32_t>(item) / per_row;
        c = (item - r * per_row) * (ROWS ? 8 : 64);
        if (!ROWS) {
            const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
            r = r * 32 + (warp & 3) * 8 + (lane >> 2);
            c += (warp >> 2) * 32 + (lane & 3) * 8;
        }
    }
};
template <typename T>
__device__ __forceinline__ void ns_load8(const T* row, int64_t c, int64_t cols, bool vec, float (&f)[8]) {
    constexpr int VEC = Elem<T>::VEC;
    if (vec && c + 8 <= cols) {
#pragma unroll
        for (int h = 0; h < 8 / VEC; h++) {
            float part[VEC];
            Elem<T>::unpack(reinterpret_cast<const uint4*>(row + c)[h], part);
#pragma unroll
            for (int i = 0; i < VEC; i++) f[h * VEC + i] = part[i];
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; i++) f[i] = c + i < cols ? Elem<T>::to(row[c + i]) : 0.f;
}

// Sums of squares in 64 bits (fp32 squares leave the range from 1.8e19 on). For the Muon step the pass also updates
// the momentum and leaves the matrix to orthogonalise in X32.
template <typename T, bool MUON>
__global__ void __launch_bounds__(256)
ns_norm_kernel(const T* g, float* momentum, float* X32, double* partial, int64_t rows, int64_t cols, int64_t ld_g,
               int64_t stride_g, int64_t ldx, int64_t stridex, float mu, int nesterov, int vec) {
    __shared__ double buf[8];
    kernel_wait_previous();
    kernel_allow_next();
    const int64_t b = blockIdx.y;
    double sum = 0.0;
#pragma unroll 4
    for (NsGroups<!MUON> it(rows, cols); it.more(); it.next()) {
        int64_t r, c;
        it.at(r, c);
        if (r >= rows || c >= cols) continue;
        float v[8];
        ns_load8(g + b * stride_g + r * ld_g, c, cols, vec, v);
        if (MUON) {
            float m[8];
            float* mp = momentum + (b * rows + r) * cols + c;
            ns_load8(const_cast<const float*>(mp - c), c, cols, vec, m);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                m[i] = fmaf(mu, m[i], v[i]);
                v[i] = nesterov ? fmaf(mu, m[i], v[i]) : m[i];
            }
            if (vec && c + 8 <= cols) {
                reinterpret_cast<float4*>(mp)[0] = make_float4(m[0], m[1], m[2], m[3]);
                reinterpret_cast<float4*>(mp)[1] = make_float4(m[4], m[5], m[6], m[7]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (c + i < cols) mp[i] = m[i];
            }
            float4* xp = reinterpret_cast<float4*>(X32 + b * stridex + ns_state_at(r, c, ldx));
            xp[0] = make_float4(v[0], v[1], v[2], v[3]);
            xp[32] = make_float4(v[4], v[5], v[6], v[7]);
        }
#pragma unroll
        for (int i = 0; i < 8; i++) sum += static_cast<double>(v[i]) * v[i];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 8; w++) sum += buf[w];
        partial[b * kNormParts + blockIdx.x] = sum;
    }
}

// X = G / (norm + eps) in both copies. Every CTA adds the partial sums itself, its first groups on their way meanwhile, and
// takes several tiles, each loaded before the one before it is written.
template <typename T, bool MUON>
__global__ void __launch_bounds__(256)
ns_start_kernel(const T* g, float* X32, __half* X16, const double* partial, int parts, int64_t rows, int64_t cols, int64_t ld_g,
                int64_t stride_g, int64_t ldx, int64_t stridex, float eps, int vec) {
    __shared__ double buf[8];
    kernel_wait_previous();
    kernel_allow_next();
    const int64_t b = blockIdx.y;
    const auto inside = [&](const NsGroups<false>& it, int64_t& r, int64_t& c) {
        if (!it.more()) return false;
        it.at(r, c);
        return r < rows && c < cols;
    };
    const auto load = [&](const NsGroups<false>& it, float (&v)[8]) {
        int64_t r, c;
        if (!inside(it, r, c)) return;
        if (MUON) {
            const float4* xp = reinterpret_cast<const float4*>(X32 + b * stridex + ns_state_at(r, c, ldx));
            const float4 lo = xp[0], hi = xp[32];
            v[0] = lo.x; v[1] = lo.y; v[2] = lo.z; v[3] = lo.w;
            v[4] = hi.x; v[5] = hi.y; v[6] = hi.z; v[7] = hi.w;
        } else {
            ns_load8(g + b * stride_g + r * ld_g, c, cols, vec, v);
        }
    };
    NsGroups<false> it(rows, cols);
    float v[8];
    load(it, v);
    double sum = 0.0;
    for (int i = threadIdx.x; i < parts; i += 256) sum += partial[b * kNormParts + i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = sum;
    __syncthreads();
    sum = 0.0;
    for (int w = 0; w < 8; w++) sum += buf[w];
    // x / (norm + eps) as x 2^-e / d, so that a norm beyond fp32's range divides too; a zero divisor leaves zeros
    int e = 0;
    const double norm = sqrt(sum) + eps;
    if (norm > 0.0 && norm <= 1.7e308) frexp(norm, &e);
    e = max(-100, min(100, e));
    const float div = norm == 0.0 ? 1.f : static_cast<float>(ldexp(norm, -e)), pre = exp2f(static_cast<float>(-e));
    while (it.more()) {
        NsGroups<false> following = it;
        following.next();
        float next_v[8];
        load(following, next_v);
        int64_t r, c;
        if (inside(it, r, c)) {
            uint32_t h[4], l[4];
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = v[i] * pre / div * kNsScale;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const __half2 two = __floats2half2_rn(v[2 * i], v[2 * i + 1]), rest = ns_low(v[2 * i], v[2 * i + 1], two);
                h[i] = *reinterpret_cast<const uint32_t*>(&two);
                l[i] = *reinterpret_cast<const uint32_t*>(&rest);
            }
            float4* xp = reinterpret_cast<float4*>(X32 + b * stridex + ns_state_at(r, c, ldx));
            xp[0] = make_float4(v[0], v[1], v[2], v[3]);
            xp[32] = make_float4(v[4], v[5], v[6], v[7]);
            // padded rows: whole groups; the low parts behind all matrices' high parts
            *reinterpret_cast<uint4*>(X16 + (b * rows + r) * ldx + c) = make_uint4(h[0], h[1], h[2], h[3]);
            *reinterpret_cast<uint4*>(X16 + ((gridDim.y + b) * rows + r) * ldx + c) = make_uint4(l[0], l[1], l[2], l[3]);
        }
        it = following;
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = next_v[i];
    }
}

// ---- host side ------------------------------------------------------------------------------------------------
// Three tile sizes, and what a k block of 64 and an epilogue cost relative to each other (cycles where the high parts
// are multiplied alone; with all three terms a block takes 1.0 us, 0.6 and 0.5, the first bound by the tensor pipe and
// shared memory, the others by their loads at 64 bytes a cycle and SM). Between two tiles of a CTA the epilogue of the
// first slows the second down (by about half its own length when it is X's, which moves twelve bytes an entry); the last
// epilogue stands alone. Large products are fastest by pairs, products of few tiles by the size that gives every SM one, the
// smallest by the tile with the shortest way (by pairs, 128 x 128 and 128 x 64: 8192 x 4096 5.8, 7.1 and 12.5 ms; 2048 x 2048
// 706, 501 and 978 us, chosen product by product 510; 256 x 512 251, 155 and 104). A = X X^T of a long X has few tiles and a
// long contraction: then several CTAs share a tile, at the price of another kernel that adds their parts (about 6000 cycles).
constexpr int kNsSms = 148;  // the workspace does not depend on the device
enum { NS_PAIR = 0, NS_SINGLE = 1, NS_SMALL = 2 };
struct NsChoice {
    int tile, splits;
};
static NsChoice ns_choose(int mode, int64_t M, int64_t N, int64_t K, int64_t batch) {
    struct { int64_t bm, bn, workers, block, epilogue; } const tile[3] = {
        {256, 256, kNsSms / 2, 565, mode == NS_APPLY ? 10000 : 6000},
        {128, 128, kNsSms, 455, mode == NS_APPLY ? 4000 : 3000},
        {128, 64, kNsSms, 390, 2500}};
    NsChoice best{0, 1};
    int64_t least = INT64_MAX;
    for (int t = 0; t < 3; t++) {
        const int64_t m = (M + tile[t].bm - 1) / tile[t].bm, n = (N + tile[t].bn - 1) / tile[t].bn, blocks = (K + 63) / 64;
        const int64_t tiles = batch * (mode != NS_APPLY && tile[t].bm == tile[t].bn ? m * (m + 1) / 2 : m * n);
        const int64_t rounds = (tiles + tile[t].workers - 1) / tile[t].workers;
        const int64_t whole = rounds * blocks * tile[t].block + (rounds - 1) * (mode == NS_APPLY ? tile[t].epilogue / 2 : 0) + tile[t].epilogue;
        if (whole < least) {
            least = whole;
            best = NsChoice{t, 1};
        }
        int64_t splits = tile[t].workers / tiles;
        if (splits > blocks / 4) splits = blocks / 4;
        if (mode != NS_GRAM || splits < 2) continue;
        const int64_t shared = (blocks + splits - 1) / splits * tile[t].block + tile[t].epilogue + 6000;
        if (shared < least) {
            least = shared;
            best = NsChoice{t, (int)splits};
        }
    }
    return best;
}

struct NsPlan {
    bool tall;
    int64_t S, L, ldx, lda, stridex;  // stridex: floats of a matrix's X32, whole blocks of 32 rows
    int splits;      // of the contraction of A
    size_t x32, x16, gram, diag, norm, part;
    size_t total() const { return x32 + 2 * x16 + 2 * gram + diag + part + norm; }
};

static int plan_ns(const nzb_orthogonalize_desc* d, NsPlan* pl) {
    if (!d) return fail(NZB_ERR_BAD_ARG, "descriptor is null");
    if (d->batch < 0 || d->rows < 0 || d->cols < 0) return fail(NZB_ERR_BAD_ARG, "negative extent");
    if (d->batch > 65535 || d->rows > (1 << 24) || d->cols > (1 << 24)) return fail(NZB_ERR_UNSUPPORTED, "batch at most 65535, sides at most 2^24");
    if (d->steps < 1 || d->steps > 64) return fail(NZB_ERR_BAD_ARG, "steps must be in [1, 64]");
    if (!(d->eps >= 0.f)) return fail(NZB_ERR_BAD_ARG, "eps is negative or NaN");
    pl->tall = d->rows > d->cols;
    pl->S = pl->tall ? d->cols : d->rows;
    pl->L = pl->tall ? d->rows : d->cols;
    if (pl->S > (1 << 20)) return fail(NZB_ERR_UNSUPPORTED, "the short side is at most 2^20");
    pl->ldx = round_up(d->cols > 0 ? d->cols : 1, kOperandKAlign);
    pl->lda = round_up(pl->S > 0 ? pl->S : 1, kOperandKAlign);
    pl->stridex = round_up(d->rows, 32) * pl->ldx;
    pl->x32 = (size_t)round_up(d->batch * pl->stridex * 4, 256);
    pl->x16 = (size_t)round_up(2 * d->batch * d->rows * pl->ldx * 2, 256);  // high and low parts
    pl->gram = (size_t)round_up(2 * d->batch * pl->S * pl->lda * 2, 256);
    pl->diag = (size_t)round_up(d->batch * pl->S * 4, 256);
    pl->norm = (size_t)(d->batch * kNormParts * 8);
    pl->splits = d->batch > 0 && pl->S > 0 ? ns_choose(NS_GRAM, pl->S, pl->S, pl->L, d->batch).splits : 1;
    pl->part = pl->splits > 1 ? (size_t)(pl->splits * d->batch * round_up(pl->S, 32) * pl->lda * 4) : 0;
    return NZB_OK;
}

template <class Cfg, int MODE>
static int launch_product(const CUtensorMap& tmA, const CUtensorMap& tmB, NsParams& p, int64_t batch, const DeviceState& ds,
                          cudaStream_t s) {
    static std::atomic<uint64_t> smem_set{0};
    const auto kernel = ns_product_kernel<Cfg, MODE>;
    int rc = ensure_dynamic_smem(smem_set, reinterpret_cast<const void*>(kernel), Cfg::SMEM_BYTES);
    if (rc != NZB_OK) return rc;
    p.tiles_m = (p.M + Cfg::BM - 1) / Cfg::BM;
    p.tiles_n = (p.N + Cfg::BN - 1) / Cfg::BN;
    p.group_m = 8;
    p.symmetric = MODE != NS_APPLY && Cfg::BM == Cfg::BN;
    p.tiles_per_matrix = p.symmetric ? (int64_t)p.tiles_m * (p.tiles_m + 1) / 2 : (int64_t)p.tiles_m * p.tiles_n;
    p.tiles = p.tiles_per_matrix * batch;
    if (p.splits < 1) p.splits = 1;
    int64_t workers = Cfg::PAIR ? ds.sm_count / 2 : ds.sm_count;
    if (p.tiles * p.splits < workers) workers = p.tiles * p.splits;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(Cfg::PAIR ? 2 * workers : workers));
    cfg.blockDim = dim3(Cfg::THREADS);
    cfg.dynamicSmemBytes = Cfg::SMEM_BYTES;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 2;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = Cfg::PAIR ? 2 : 1;
    NZB_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, tmA, tmB, p));
    return NZB_OK;
}

// A product's operand of the whole batch: `rows` x `cols` halves, the contraction along the row or down the rows;
// `box`: rows of the tile that a load brings (K-major).
static int operand(CUtensorMap* map, const __half* base, bool mn, int64_t rows, int64_t cols, int64_t ld, int64_t batch, int box) {
    return mn ? make_operand_map_mn(map, base, rows, cols, ld, batch) : make_operand_map(map, base, cols, ld, rows, batch, box);
}
struct NsOperand {
    const __half* base;
    bool mn;
    int64_t rows, cols, ld;
};
template <class Cfg, int MODE>
static int launch_product_of(const NsOperand& a, const NsOperand& b, NsParams& p, int64_t batch, const DeviceState& ds, cudaStream_t s) {
    CUtensorMap tmA, tmB;
    int rc = operand(&tmA, a.base, a.mn, a.rows, a.cols, a.ld, 2 * batch, 128);
    if (rc == NZB_OK) rc = operand(&tmB, b.base, b.mn, b.rows, b.cols, b.ld, 2 * batch, Cfg::B_ROWS);
    p.a_mn = a.mn;
    p.b_mn = b.mn;
    return rc == NZB_OK ? launch_product<Cfg, MODE>(tmA, tmB, p, batch, ds, s) : rc;
}
template <int MODE>
static int launch_best(const NsOperand& a, const NsOperand& b, NsParams& p, int64_t K, int64_t batch, const DeviceState& ds, cudaStream_t s) {
    p.k_blocks = (int32_t)((K + 63) / 64);
    p.last_ksteps = (int32_t)((K - (int64_t)(p.k_blocks - 1) * 64 + 15) / 16);
    const NsChoice c = ns_choose(MODE, p.M, p.N, K, batch);
    p.splits = c.splits;
    p.batch = batch;
    if (c.tile == NS_PAIR) return launch_product_of<NsCfg<true, 256>, MODE>(a, b, p, batch, ds, s);
    if (c.tile == NS_SINGLE) return launch_product_of<NsCfg<false, 128>, MODE>(a, b, p, batch, ds, s);
    return launch_product_of<NsCfg<false, 64>, MODE>(a, b, p, batch, ds, s);
}

struct NsTarget {
    int kind;
    void* out;
    int64_t ld, stride;
    float w_keep, w_step;
};

static int run_ns(const nzb_orthogonalize_desc* d, const NsPlan& pl, uint8_t* ws, const NsTarget& target, const DeviceState& ds,
                  cudaStream_t s) {
    float* X32 = reinterpret_cast<float*>(ws);
    __half* X16[2] = {reinterpret_cast<__half*>(ws + pl.x32), reinterpret_cast<__half*>(ws + pl.x32 + pl.x16)};
    __half* A16 = reinterpret_cast<__half*>(ws + pl.x32 + 2 * pl.x16);
    __half* B16 = reinterpret_cast<__half*>(ws + pl.x32 + 2 * pl.x16 + pl.gram);
    float* diag = reinterpret_cast<float*>(ws + pl.x32 + 2 * pl.x16 + 2 * pl.gram);
    const NsOperand gram{A16, false, pl.S, pl.S, pl.lda}, poly{B16, false, pl.S, pl.S, pl.lda};
    int rc;
    float* partial = reinterpret_cast<float*>(ws + pl.x32 + 2 * pl.x16 + 2 * pl.gram + pl.diag);
    for (int step = 0; step < d->steps; step++) {
        const int cur = step & 1;
        NsParams p{};
        p.c0 = d->coef[0]; p.c1 = d->coef[1]; p.c2 = d->coef[2];
        p.diag = diag;
        p.short_side = pl.S;
        p.status = ds.status_dev;
        // A = X X^T, or X^T X of a tall matrix
        p.M = p.N = (int32_t)pl.S;
        p.out16 = A16;
        p.ld16 = pl.lda;
        p.stride16 = pl.S * pl.lda;
        p.low16 = d->batch * p.stride16;
        p.partial = partial;
        p.stride_part = round_up(pl.S, 32) * pl.lda;
        const NsOperand x_k{X16[cur], false, d->rows, d->cols, pl.ldx}, x_mn{X16[cur], true, d->rows, d->cols, pl.ldx};
        rc = launch_best<NS_GRAM>(pl.tall ? x_mn : x_k, pl.tall ? x_mn : x_k, p, pl.L, d->batch, ds, s);
        if (rc != NZB_OK) return rc;
        if (p.splits > 1) {
            const int64_t side = (pl.S + 31) / 32, warps = d->batch * side * (side + 1) / 2;
            NZB_CUDA_TRY(launch_programmatic(ns_gram_sum_kernel, (unsigned)((warps + 3) / 4), 128, 0, s, p));
        }
        // B = c1 A + c2 A A; A is symmetric, so both operands are read along its rows
        p.out16 = B16;
        p.gram = A16;
        rc = launch_best<NS_POLY>(gram, gram, p, pl.S, d->batch, ds, s);
        if (rc != NZB_OK) return rc;
        // X = c0 X + B X, or c0 X + X B
        p.M = (int32_t)d->rows;
        p.N = (int32_t)d->cols;
        p.by_column = pl.tall;
        p.out16 = X16[cur ^ 1];
        p.ld16 = p.ldx = pl.ldx;
        p.stride16 = d->rows * pl.ldx;
        p.low16 = d->batch * p.stride16;
        p.stridex = pl.stridex;
        p.X32 = X32;
        if (step == d->steps - 1) {
            const int64_t size = target.kind == NS_OUT_F16 || target.kind == NS_OUT_BF16 ? 2 : 4;
            p.out_kind = target.kind;
            p.out = target.out;
            p.ld_out = target.ld;
            p.stride_out = target.stride;
            p.out_vec = aligned_to(target.out, 16) && target.ld * size % 16 == 0 && target.stride * size % 16 == 0;
            p.w_keep = target.w_keep;
            p.w_step = target.w_step;
        }
        rc = launch_best<NS_APPLY>(pl.tall ? x_k : poly, pl.tall ? poly : x_mn, p, pl.S, d->batch, ds, s);
        if (rc != NZB_OK) return rc;
    }
    return NZB_OK;
}

static int check_ws(const NsPlan& pl, const void* ws, size_t bytes) {
    if (!ws || bytes < pl.total()) return fail(NZB_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", pl.total(), ws ? bytes : (size_t)0);
    if (!aligned_to(ws, 256)) return fail(NZB_ERR_WORKSPACE, "workspace must be 256-byte aligned");
    return NZB_OK;
}

// The two elementwise passes: CTAs of 256 threads per matrix. A few per SM over the whole batch, so that what each does
// once (the sums' joins in 64 bits) does not outweigh its share: 4 x 1000 x 1400 bf16 244.7 -> 238.5 us against a CTA per 2048
// elements, 256 x 512 fp32 80.9 -> 77.0.
template <typename T, bool MUON>
static int launch_start(const nzb_orthogonalize_desc* d, const NsPlan& pl, uint8_t* ws, const T* g, float* momentum, int64_t ld_g,
                        int64_t stride_g, float mu, int nesterov, int vec, cudaStream_t s) {
    float* X32 = reinterpret_cast<float*>(ws);
    __half* X16 = reinterpret_cast<__half*>(ws + pl.x32);
    double* partial = reinterpret_cast<double*>(ws + pl.total() - pl.norm);
    const int64_t tiles = ((d->rows + 31) / 32) * ((d->cols + 63) / 64);
    const auto ctas = [&](int64_t all) {
        const int64_t each = (all + d->batch - 1) / d->batch;
        return (unsigned)(each < tiles ? each : tiles);
    };
    const unsigned parts = ctas(kNormParts);
    NZB_CUDA_TRY(launch_programmatic(ns_norm_kernel<T, MUON>, dim3(parts, (unsigned)d->batch), 256, 0, s, g, momentum, X32, partial, d->rows,
                                     d->cols, ld_g, stride_g, pl.ldx, pl.stridex, mu, nesterov, vec));
    NZB_CUDA_TRY(launch_programmatic(ns_start_kernel<T, MUON>, dim3(ctas(std::max<int64_t>(6 * kNsSms, tiles * d->batch / 8)), (unsigned)d->batch), 256, 0, s, g, X32, X16, partial,
                                     (int)parts, d->rows, d->cols, ld_g, stride_g, pl.ldx, pl.stridex, d->eps, vec));
    return NZB_OK;
}

}  // namespace nzb

using namespace nzb;

extern "C" {

int nzb_orthogonalize_workspace_bytes(const nzb_orthogonalize_desc* d, size_t* bytes_out) {
    if (!bytes_out) return fail(NZB_ERR_BAD_ARG, "bytes_out is null");
    NsPlan pl;
    int rc = plan_ns(d, &pl);
    if (rc != NZB_OK) return rc;
    *bytes_out = pl.total();
    return NZB_OK;
}

int nzb_orthogonalize(const nzb_orthogonalize_desc* d, const void* g, void* out, void* workspace, size_t workspace_bytes,
                      void* stream) {
    NsPlan pl;
    int rc = plan_ns(d, &pl);
    if (rc != NZB_OK) return rc;
    if (!known_dtype(d->dtype) || !known_dtype(d->out_dtype)) return fail(NZB_ERR_BAD_ARG, "unknown element type");
    if (d->ld_g < d->cols || d->ld_out < d->cols) return fail(NZB_ERR_BAD_ARG, "leading dimension smaller than the row length");
    if (d->batch == 0 || d->rows == 0 || d->cols == 0) return NZB_OK;
    if (d->batch > 1 && d->stride_out < d->cols) return fail(NZB_ERR_BAD_ARG, "output matrices overlap");
    if (!g || !out) return fail(NZB_ERR_BAD_ARG, "g and out must be non-null");
    if (!aligned_to(g, dtype_size(d->dtype)) || !aligned_to(out, dtype_size(d->out_dtype)))
        return fail(NZB_ERR_BAD_ARG, "pointer is not a multiple of its element's size");
    rc = check_ws(pl, workspace, workspace_bytes);
    if (rc != NZB_OK) return rc;
    DeviceState* ds;
    rc = get_device_state(&ds);
    if (rc != NZB_OK) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    const int64_t size = dtype_size(d->dtype);
    const int vec = aligned_to(g, 16) && d->ld_g * size % 16 == 0 && (d->batch == 1 || d->stride_g * size % 16 == 0);
    NZB_DISPATCH_DTYPE(d->dtype, T, {
        rc = launch_start<T, false>(d, pl, ws, static_cast<const T*>(g), nullptr, d->ld_g, d->stride_g, 0.f, 0, vec, s);
    });
    if (rc != NZB_OK) return rc;
    const int kind = d->out_dtype == NZB_F32 ? NS_OUT_F32 : d->out_dtype == NZB_F16 ? NS_OUT_F16 : NS_OUT_BF16;
    return run_ns(d, pl, ws, NsTarget{kind, out, d->ld_out, d->stride_out, 0.f, 0.f}, *ds, s);
}

int nzb_muon_workspace_bytes(const nzb_orthogonalize_desc* d, size_t* bytes_out) {
    return nzb_orthogonalize_workspace_bytes(d, bytes_out);
}

int nzb_muon(const nzb_orthogonalize_desc* d, float* w, float* momentum, const float* grad, float lr, float scale, float mu,
             float weight_decay, int nesterov, void* workspace, size_t workspace_bytes, void* stream) {
    NsPlan pl;
    int rc = plan_ns(d, &pl);
    if (rc != NZB_OK) return rc;
    if (d->batch == 0 || d->rows == 0 || d->cols == 0) return NZB_OK;
    if (!w || !momentum || !grad) return fail(NZB_ERR_BAD_ARG, "w, momentum and grad must be non-null");
    if (w == momentum || grad == momentum) return fail(NZB_ERR_BAD_ARG, "momentum needs memory of its own");
    if (!aligned_to(w, 4) || !aligned_to(momentum, 4) || !aligned_to(grad, 4))
        return fail(NZB_ERR_BAD_ARG, "pointer is not a multiple of its element's size");
    rc = check_ws(pl, workspace, workspace_bytes);
    if (rc != NZB_OK) return rc;
    DeviceState* ds;
    rc = get_device_state(&ds);
    if (rc != NZB_OK) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    const int64_t n = d->rows * d->cols;
    const int vec = aligned_to(grad, 16) && aligned_to(momentum, 16) && d->cols % 4 == 0;
    rc = launch_start<float, true>(d, pl, ws, grad, momentum, d->cols, n, mu, nesterov, vec, s);
    if (rc != NZB_OK) return rc;
    return run_ns(d, pl, ws, NsTarget{NS_OUT_WEIGHT, w, d->cols, n, 1.f - lr * weight_decay, lr * scale}, *ds, s);
}

}  // extern "C"
