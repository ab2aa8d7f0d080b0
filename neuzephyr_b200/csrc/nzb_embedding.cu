// Rows of a table by token number, and the gradient of the table. Beside Linear's forward and weight gradient:
// the same products with a one-hot left operand, done as copies and as sums over sorted tokens.
//
// Backward: dW[v] = scale * sum_{t: id_t = v} dy[t]. Atomics would add in an order that changes from run to run,
// so the tokens are sorted first (stable, by token number) and every row is summed in the order of t:
//   1. one CTA per tile of 16384 tokens sorts the tile in shared memory (radix, up to 9 bits a pass; the items
//      wait in registers between passes, so one copy of the keys is enough) and cuts the runs of equal tokens
//      into pieces of at most 64;
//   2. one warp per piece and 32 vectors of columns sums the piece's rows; a run of one piece goes straight to
//      the table, the pieces of a longer one to the workspace;
//   3. the pieces of the longer runs are added in order.
// Tiles after the first add to the rows the earlier ones wrote, in launch order: the same bits every time.
#include "nzb_internal.h"
#include "nzb_elem.cuh"

namespace nzb {

constexpr int kSortTile = 16384;
constexpr int kSortThreads = 1024;
constexpr int kSortItems = kSortTile / kSortThreads;
constexpr int kSortMaxBins = 512;
constexpr int kPiece = 64;                                  // tokens summed by one warp
constexpr int kMaxSlots = 2 * (kSortTile / kPiece);         // pieces of runs longer than kPiece, per tile

// What the sort leaves for the sums, per tile.
struct SortTile {
    int32_t pieces, runs;                 // runs: those of more than one piece
    int32_t order[kSortTile];             // token positions within the tile, sorted
    int32_t piece_start[kSortTile + 1];
    int32_t piece_key[kSortTile];
    int32_t piece_slot[kSortTile];        // partial sum's row, or -1: the piece is a whole run
    int32_t run_key[kSortTile / kPiece + 1];
    int32_t run_slot[kSortTile / kPiece + 2];  // first partial row; the next run's start is its end
};

struct SortSmem {
    uint32_t key[kSortTile];
    uint32_t hist[32][kSortMaxBins];
    uint32_t bin_base[kSortMaxBins];
    uint16_t pos[kSortTile];
    int32_t scan[32];
    int32_t scan2[32];
    int32_t scan3[32];
};

__device__ __forceinline__ int32_t warp_inclusive_sum(int32_t v, int lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int32_t u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    return v;
}
__device__ __forceinline__ int32_t warp_inclusive_max(int32_t v, int lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int32_t u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v = max(v, u);
    }
    return v;
}

template <typename Index>
__global__ void __launch_bounds__(kSortThreads, 1)
embedding_sort_kernel(const Index* __restrict__ index, int64_t tokens, int64_t vocab, int64_t padding, int digit_bits,
                      int passes, SortTile* __restrict__ out_tiles, uint32_t* __restrict__ present) {
    extern __shared__ uint4 smem_sort[];
    SortSmem& s = *reinterpret_cast<SortSmem*>(smem_sort);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t t0 = static_cast<int64_t>(blockIdx.x) * kSortTile;
    const int count = static_cast<int>(min(static_cast<int64_t>(kSortTile), tokens - t0));
    SortTile& out = out_tiles[blockIdx.x];
    const uint32_t none = static_cast<uint32_t>(vocab);  // sorts behind every token

    uint32_t k[kSortItems];
    uint16_t p[kSortItems];
#pragma unroll
    for (int i = 0; i < kSortItems; i++) {
        const int at = warp * (kSortTile / 32) + i * 32 + lane;
        uint32_t key = none;
        if (at < count) {
            const int64_t v = static_cast<int64_t>(index[t0 + at]);
            if (v >= 0 && v < vocab && v != padding) {
                key = static_cast<uint32_t>(v);
                if (blockIdx.x == 0) atomicOr(present + (key >> 5), 1u << (key & 31));
            }
        }
        k[i] = key;
        p[i] = static_cast<uint16_t>(at);
    }

    const int bins = 1 << digit_bits;
    const uint32_t mask = bins - 1;
    for (int pass = 0; pass < passes; pass++) {
        const int shift = pass * digit_bits;
        for (int i = lane; i < bins; i += 32) s.hist[warp][i] = 0;
        __syncwarp();
        uint32_t rank[kSortItems];
#pragma unroll
        for (int i = 0; i < kSortItems; i++) {
            const uint32_t d = (k[i] >> shift) & mask;
            const uint32_t peers = __match_any_sync(0xffffffffu, d);
            const int leader = __ffs(peers) - 1;
            uint32_t before = 0;
            if (lane == leader) {
                before = s.hist[warp][d];
                s.hist[warp][d] = before + __popc(peers);
            }
            before = __shfl_sync(0xffffffffu, before, leader);
            rank[i] = before + __popc(peers & ((1u << lane) - 1));
            __syncwarp();
        }
        __syncthreads();
        // exclusive over the warps within a bin, then over the bins
        uint32_t total = 0;
        if (tid < bins) {
#pragma unroll 8
            for (int w = 0; w < 32; w++) {
                const uint32_t c = s.hist[w][tid];
                s.hist[w][tid] = total;
                total += c;
            }
        }
        const int32_t incl = warp_inclusive_sum(static_cast<int32_t>(total), lane);
        if (lane == 31) s.scan[warp] = incl;
        __syncthreads();
        if (warp == 0) s.scan[lane] = warp_inclusive_sum(s.scan[lane], lane);
        __syncthreads();
        if (tid < bins) s.bin_base[tid] = static_cast<uint32_t>(incl) - total + (warp > 0 ? s.scan[warp - 1] : 0);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kSortItems; i++) {
            const uint32_t d = (k[i] >> shift) & mask;
            const uint32_t to = s.bin_base[d] + s.hist[warp][d] + rank[i];
            s.key[to] = k[i];
            s.pos[to] = p[i];
        }
        __syncthreads();
        if (pass + 1 < passes) {
#pragma unroll
            for (int i = 0; i < kSortItems; i++) {
                const int at = warp * (kSortTile / 32) + i * 32 + lane;
                k[i] = s.key[at];
                p[i] = s.pos[at];
            }
            __syncthreads();
        }
    }
    for (int i = tid; i < count; i += kSortThreads) out.order[i] = s.pos[i];

    // runs of equal tokens and their pieces: every thread looks at kSortItems neighbours
    const int i0 = tid * kSortItems;
    int32_t last_head = -1;
#pragma unroll
    for (int i = 0; i < kSortItems; i++) {
        const int at = i0 + i;
        if (at == 0 || s.key[at] != s.key[at - 1]) last_head = at;
    }
    const int32_t head_incl = warp_inclusive_max(last_head, lane);
    if (lane == 31) s.scan[warp] = head_incl;
    __syncthreads();
    if (warp == 0) s.scan[lane] = warp_inclusive_max(s.scan[lane], lane);
    __syncthreads();
    int32_t head = __shfl_up_sync(0xffffffffu, head_incl, 1);
    if (lane == 0) head = -1;
    if (warp > 0) head = max(head, s.scan[warp - 1]);
    const int32_t head0 = head;
    int32_t n_piece = 0, n_slot = 0, n_run = 0;
#pragma unroll
    for (int i = 0; i < kSortItems; i++) {
        const int at = i0 + i;
        if (at == 0 || s.key[at] != s.key[at - 1]) head = at;
        if (s.key[at] != none && (at - head) % kPiece == 0) {
            n_piece++;
            if (head + kPiece < kSortTile && s.key[head + kPiece] == s.key[at]) {
                n_slot++;
                if (at == head) n_run++;
            }
        }
    }
    const int32_t ip = warp_inclusive_sum(n_piece, lane), is = warp_inclusive_sum(n_slot, lane), ir = warp_inclusive_sum(n_run, lane);
    __syncthreads();
    if (lane == 31) {
        s.scan[warp] = ip;
        s.scan2[warp] = is;
        s.scan3[warp] = ir;
    }
    __syncthreads();
    if (warp == 0) {
        s.scan[lane] = warp_inclusive_sum(s.scan[lane], lane);
        s.scan2[lane] = warp_inclusive_sum(s.scan2[lane], lane);
        s.scan3[lane] = warp_inclusive_sum(s.scan3[lane], lane);
    }
    __syncthreads();
    int32_t piece = ip - n_piece + (warp > 0 ? s.scan[warp - 1] : 0);
    int32_t slot = is - n_slot + (warp > 0 ? s.scan2[warp - 1] : 0);
    int32_t run = ir - n_run + (warp > 0 ? s.scan3[warp - 1] : 0);
    head = head0;
#pragma unroll
    for (int i = 0; i < kSortItems; i++) {
        const int at = i0 + i;
        if (at == 0 || s.key[at] != s.key[at - 1]) {
            if (s.key[at] == none) out.piece_start[piece] = at;  // end of the last piece: one thread gets here
            head = at;
        }
        if (s.key[at] != none && (at - head) % kPiece == 0) {
            const bool longer = head + kPiece < kSortTile && s.key[head + kPiece] == s.key[at];
            out.piece_start[piece] = at;
            out.piece_key[piece] = static_cast<int32_t>(s.key[at]);
            out.piece_slot[piece] = longer ? slot : -1;
            if (longer && at == head) {
                out.run_key[run] = static_cast<int32_t>(s.key[at]);
                out.run_slot[run] = slot;
                run++;
            }
            if (longer) slot++;
            piece++;
        }
    }
    if (tid == kSortThreads - 1) {
        out.pieces = piece;
        out.runs = run;
        out.run_slot[run] = slot;
        if (s.key[kSortTile - 1] != none) out.piece_start[piece] = kSortTile;
    }
}

// Columns c .. c + VEC - 1 (vector form) of a gradient row.
template <int VEC>
__device__ __forceinline__ void put_columns(float* row, int64_t c, int64_t dim, const float (&acc)[VEC], bool add, bool vec) {
    if (vec && c + VEC <= dim) {
#pragma unroll
        for (int i = 0; i < VEC; i += 4) {
            float4 v = make_float4(acc[i], acc[i + 1], acc[i + 2], acc[i + 3]);
            float4* at = reinterpret_cast<float4*>(row + c + i);
            if (add) {
                const float4 o = *at;
                v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
            }
            *at = v;
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < VEC; i++)
        if (c + i < dim) row[c + i] = add ? row[c + i] + acc[i] : acc[i];
}

template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(256)
embedding_sum_kernel(const T* __restrict__ dy, const SortTile* __restrict__ tile, const uint32_t* __restrict__ present,
                     float* __restrict__ dtable, float* __restrict__ partial, int64_t vocab, int64_t dim, int64_t ld_table,
                     int64_t ld_y, float scale, int add, int zero_rest, int vec_out) {
    constexpr int VEC = Elem<T>::VEC;
    const int lane = threadIdx.x & 31;
    const int64_t warp = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
    const int64_t warps = (static_cast<int64_t>(gridDim.x) * blockDim.x) >> 5;
    const int64_t blocks = (dim + 32 * VEC - 1) / (32 * VEC);  // column blocks of a row
    const int64_t items = tile->pieces * blocks;
    for (int64_t item = warp; item < items; item += warps) {
        const int64_t piece = item / blocks, c0 = (item - piece * blocks) * 32 * VEC;
        const int i0 = tile->piece_start[piece], i1 = tile->piece_start[piece + 1];
        const int slot = tile->piece_slot[piece];
        float acc[VEC];
#pragma unroll
        for (int i = 0; i < VEC; i++) acc[i] = 0.f;
        const int64_t c = ALIGNED ? c0 + lane * VEC : c0 + lane;
        for (int i = i0; i < i1; i++) {
            const T* row = dy + static_cast<int64_t>(tile->order[i]) * ld_y;
            if (ALIGNED) {
                float f[VEC];
                if (c < dim) {
                    Elem<T>::unpack(load_block(row, c, dim), f);
#pragma unroll
                    for (int j = 0; j < VEC; j++) acc[j] += f[j];
                }
            } else {
#pragma unroll
                for (int j = 0; j < VEC; j++)
                    if (c + j * 32 < dim) acc[j] += Elem<T>::to(row[c + j * 32]);
            }
        }
        const bool whole = slot < 0;
        float* to = whole ? dtable + static_cast<int64_t>(tile->piece_key[piece]) * ld_table : partial + static_cast<int64_t>(slot) * dim;
        if (whole) {
#pragma unroll
            for (int j = 0; j < VEC; j++) acc[j] *= scale;
        }
        if (ALIGNED) {
            if (c < dim) put_columns<VEC>(to, c, dim, acc, whole && add, whole ? vec_out : dim % 4 == 0);
        } else {
#pragma unroll
            for (int j = 0; j < VEC; j++)
                if (c + j * 32 < dim) to[c + j * 32] = whole && add ? to[c + j * 32] + acc[j] : acc[j];
        }
    }
    if (!zero_rest) return;
    const float zero[4] = {0.f, 0.f, 0.f, 0.f};
    for (int64_t v = warp; v < vocab; v += warps) {
        if (present[v >> 5] >> (v & 31) & 1) continue;
        float* row = dtable + v * ld_table;
        for (int64_t c = lane * 4; c < dim; c += 128) put_columns<4>(row, c, dim, zero, false, vec_out);
    }
}

__global__ void __launch_bounds__(256)
embedding_join_kernel(const SortTile* __restrict__ tile, const float* __restrict__ partial, float* __restrict__ dtable,
                      int64_t dim, int64_t ld_table, float scale, int add) {
    const int runs = tile->runs;
    const int64_t blocks = (dim + 255) / 256;
    for (int64_t item = blockIdx.x; item < runs * blocks; item += gridDim.x) {
        const int64_t run = item / blocks;
        const int64_t c = (item - run * blocks) * 256 + threadIdx.x;
        if (c >= dim) continue;
        const int s0 = tile->run_slot[run], s1 = tile->run_slot[run + 1];
        float acc = 0.f;
        for (int s = s0; s < s1; s++) acc += partial[static_cast<int64_t>(s) * dim + c];
        float* to = dtable + static_cast<int64_t>(tile->run_key[run]) * ld_table + c;
        *to = add ? *to + scale * acc : scale * acc;
    }
}

// One 16-byte block of y per item, a few items per thread for loads in flight. ALIGNED: all rows of the table
// and of y start on 16 bytes; otherwise an item is one element.
template <typename Tab, typename Out, typename Index, bool ALIGNED>
__global__ void __launch_bounds__(256)
embedding_kernel(const Tab* __restrict__ table, const Index* __restrict__ index, Out* __restrict__ y, int64_t tokens,
                 int64_t vocab, int64_t dim, int64_t ld_table, int64_t ld_y, float scale) {
    constexpr int VEC = ALIGNED ? Elem<Out>::VEC : 1;
    const int64_t per_row = (dim + VEC - 1) / VEC;
    const int64_t items = tokens * per_row;
    const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x;
    for (int64_t item = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; item < items; item += step) {
        const int64_t t = item / per_row, c = (item - t * per_row) * VEC;
        const int64_t v = static_cast<int64_t>(index[t]);
        const bool inside = v >= 0 && v < vocab;
        const Tab* from = table + (inside ? v : 0) * ld_table;
        Out* to = y + t * ld_y;
        if (ALIGNED) {
            float f[Elem<Out>::VEC];
#pragma unroll
            for (int i = 0; i < Elem<Out>::VEC; i++) f[i] = 0.f;
            if (inside) {
                constexpr int TV = Elem<Tab>::VEC;
#pragma unroll
                for (int h = 0; h < Elem<Out>::VEC / TV; h++) {
                    float part[TV];
                    Elem<Tab>::unpack(load_block(from, c + h * TV, dim), part);
#pragma unroll
                    for (int i = 0; i < TV; i++) f[h * TV + i] = part[i] * scale;
                }
            }
            store_block(to, c, dim, Elem<Out>::pack(f));
        } else {
            to[c] = Elem<Out>::from(inside ? Elem<Tab>::to(from[c]) * scale : 0.f);
        }
    }
}

static int check_embedding(const nzb_embedding_desc* d, bool backward) {
    if (!d) return fail(NZB_ERR_BAD_ARG, "descriptor is null");
    if (d->tokens < 0 || d->vocab < 0 || d->dim < 0) return fail(NZB_ERR_BAD_ARG, "negative extent");
    if (!known_dtype(d->dtype) || !known_dtype(d->table_dtype)) return fail(NZB_ERR_BAD_ARG, "unknown element type");
    if (d->index_type != NZB_I32 && d->index_type != NZB_I64) return fail(NZB_ERR_BAD_ARG, "unknown index type");
    if (d->ld_table < d->dim || d->ld_y < d->dim) return fail(NZB_ERR_BAD_ARG, "leading dimension smaller than the row length");
    if (!backward && d->table_dtype != d->dtype && d->table_dtype != NZB_F32)
        return fail(NZB_ERR_UNSUPPORTED, "the table is fp32 or of the output's type");
    if (d->vocab >= INT32_MAX || d->dim > (1 << 24) || d->tokens > INT32_MAX)
        return fail(NZB_ERR_UNSUPPORTED, "vocab and tokens must be below 2^31, dim at most 2^24");
    return NZB_OK;
}

struct EmbeddingPlan {
    int64_t tiles;
    size_t tiles_bytes, present_bytes, partial_bytes;
    size_t total() const { return tiles_bytes + present_bytes + partial_bytes; }
};
static EmbeddingPlan plan_embedding(const nzb_embedding_desc* d) {
    EmbeddingPlan pl;
    pl.tiles = (d->tokens + kSortTile - 1) / kSortTile;
    if (pl.tiles < 1) pl.tiles = 1;
    pl.tiles_bytes = (size_t)round_up(pl.tiles * (int64_t)sizeof(SortTile), 256);
    pl.present_bytes = (size_t)round_up((d->vocab + 31) / 32 * 4, 256);
    // a run has more than one piece from kPiece + 1 tokens on
    int64_t slots = 2 * (d->tokens / kPiece);
    if (slots > kMaxSlots) slots = kMaxSlots;
    pl.partial_bytes = (size_t)round_up(slots * d->dim * 4, 256);
    return pl;
}

template <typename Tab, typename Out, typename Index>
static int launch_embedding(const nzb_embedding_desc* d, const void* table, const void* index, void* y, int sm_count,
                            cudaStream_t s) {
    const bool aligned = aligned_to(table, 16) && aligned_to(y, 16) && d->ld_table * (int64_t)sizeof(Tab) % 16 == 0 &&
                         d->ld_y * (int64_t)sizeof(Out) % 16 == 0;
    const int64_t items = d->tokens * (aligned ? (d->dim + Elem<Out>::VEC - 1) / Elem<Out>::VEC : d->dim);
    int64_t blocks = (items + 255) / 256;
    if (blocks > (int64_t)sm_count * 64) blocks = (int64_t)sm_count * 64;
    const Tab* tp = static_cast<const Tab*>(table);
    const Index* ip = static_cast<const Index*>(index);
    Out* yp = static_cast<Out*>(y);
    if (aligned)
        embedding_kernel<Tab, Out, Index, true><<<(unsigned)blocks, 256, 0, s>>>(tp, ip, yp, d->tokens, d->vocab, d->dim, d->ld_table, d->ld_y, d->scale);
    else
        embedding_kernel<Tab, Out, Index, false><<<(unsigned)blocks, 256, 0, s>>>(tp, ip, yp, d->tokens, d->vocab, d->dim, d->ld_table, d->ld_y, d->scale);
    NZB_CUDA_TRY(cudaGetLastError());
    return NZB_OK;
}

template <typename Index>
static int launch_sort(const nzb_embedding_desc* d, const void* index, const EmbeddingPlan& pl, SortTile* tiles,
                       uint32_t* present, cudaStream_t s) {
    static std::atomic<uint64_t> smem_set{0};
    int rc = ensure_dynamic_smem(smem_set, reinterpret_cast<const void*>(embedding_sort_kernel<Index>), sizeof(SortSmem));
    if (rc != NZB_OK) return rc;
    int bits = 1;
    while (d->vocab >> bits) bits++;  // vocab itself stands for "no token"
    const int passes = (bits + 8) / 9, digit = (bits + passes - 1) / passes;
    embedding_sort_kernel<Index><<<(unsigned)pl.tiles, kSortThreads, sizeof(SortSmem), s>>>(
        static_cast<const Index*>(index), d->tokens, d->vocab, d->padding_index, digit, passes, tiles, present);
    NZB_CUDA_TRY(cudaGetLastError());
    return NZB_OK;
}

}  // namespace nzb

using namespace nzb;

extern "C" {

int nzb_embedding_forward(const nzb_embedding_desc* d, const void* table, const void* index, void* y, void* stream) {
    int rc = check_embedding(d, false);
    if (rc != NZB_OK) return rc;
    if (d->tokens == 0 || d->dim == 0) return NZB_OK;
    if ((!table && d->vocab > 0) || !index || !y) return fail(NZB_ERR_BAD_ARG, "table, index and y must be non-null");
    if (!aligned_to(table, dtype_size(d->table_dtype)) || !aligned_to(y, dtype_size(d->dtype)))
        return fail(NZB_ERR_BAD_ARG, "pointer is not a multiple of its element's size");
    DeviceState* ds;
    rc = get_device_state(&ds);
    if (rc != NZB_OK) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool wide = d->index_type == NZB_I64;
    NZB_DISPATCH_DTYPE(d->dtype, Out, {
        if (d->table_dtype == d->dtype)
            rc = wide ? launch_embedding<Out, Out, int64_t>(d, table, index, y, ds->sm_count, s)
                      : launch_embedding<Out, Out, int32_t>(d, table, index, y, ds->sm_count, s);
        else
            rc = wide ? launch_embedding<float, Out, int64_t>(d, table, index, y, ds->sm_count, s)
                      : launch_embedding<float, Out, int32_t>(d, table, index, y, ds->sm_count, s);
    });
    return rc;
}

int nzb_embedding_backward_workspace_bytes(const nzb_embedding_desc* d, size_t* bytes_out) {
    if (!bytes_out) return fail(NZB_ERR_BAD_ARG, "bytes_out is null");
    int rc = check_embedding(d, true);
    if (rc != NZB_OK) return rc;
    *bytes_out = plan_embedding(d).total();
    return NZB_OK;
}

int nzb_embedding_backward(const nzb_embedding_desc* d, const void* dy, const void* index, float* dtable, void* workspace,
                           size_t workspace_bytes, void* stream) {
    int rc = check_embedding(d, true);
    if (rc != NZB_OK) return rc;
    if (d->vocab == 0 || d->dim == 0 || (d->tokens == 0 && !d->overwrite)) return NZB_OK;
    if (!dtable || (d->tokens > 0 && (!dy || !index))) return fail(NZB_ERR_BAD_ARG, "dy, index and dtable must be non-null");
    if (!aligned_to(dy, dtype_size(d->dtype)) || !aligned_to(dtable, 4))
        return fail(NZB_ERR_BAD_ARG, "pointer is not a multiple of its element's size");
    const EmbeddingPlan pl = plan_embedding(d);
    if (!workspace || workspace_bytes < pl.total())
        return fail(NZB_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", pl.total(), workspace ? workspace_bytes : (size_t)0);
    if (!aligned_to(workspace, 256)) return fail(NZB_ERR_WORKSPACE, "workspace must be 256-byte aligned");
    DeviceState* ds;
    rc = get_device_state(&ds);
    if (rc != NZB_OK) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    uint8_t* base = static_cast<uint8_t*>(workspace);
    SortTile* tiles = reinterpret_cast<SortTile*>(base);
    uint32_t* present = reinterpret_cast<uint32_t*>(base + pl.tiles_bytes);
    float* partial = reinterpret_cast<float*>(base + pl.tiles_bytes + pl.present_bytes);
    NZB_CUDA_TRY(cudaMemsetAsync(present, 0, pl.present_bytes, s));
    rc = d->index_type == NZB_I64 ? launch_sort<int64_t>(d, index, pl, tiles, present, s)
                                  : launch_sort<int32_t>(d, index, pl, tiles, present, s);
    if (rc != NZB_OK) return rc;
    const int vec_out = aligned_to(dtable, 16) && d->ld_table % 4 == 0;
    const unsigned grid = (unsigned)ds->sm_count * 8;
    for (int64_t t = 0; t < pl.tiles; t++) {
        const int add = t > 0 || !d->overwrite, zero_rest = t == 0 && d->overwrite;
        NZB_DISPATCH_DTYPE(d->dtype, T, {
            const T* from = static_cast<const T*>(dy) + t * kSortTile * d->ld_y;
            if (aligned_to(dy, 16) && d->ld_y * (int64_t)sizeof(T) % 16 == 0)
                embedding_sum_kernel<T, true><<<grid, 256, 0, s>>>(from, tiles + t, present, dtable, partial, d->vocab, d->dim, d->ld_table, d->ld_y, d->scale, add, zero_rest, vec_out);
            else
                embedding_sum_kernel<T, false><<<grid, 256, 0, s>>>(from, tiles + t, present, dtable, partial, d->vocab, d->dim, d->ld_table, d->ld_y, d->scale, add, zero_rest, vec_out);
        });
        if (d->tokens - t * kSortTile > kPiece)
            embedding_join_kernel<<<grid, 256, 0, s>>>(tiles + t, partial, dtable, d->dim, d->ld_table, d->scale, add);
        NZB_CUDA_TRY(cudaGetLastError());
    }
    return NZB_OK;
}

}  // extern "C"
