// Rows of a table by token number, and the gradient of the table. Beside Linear's forward and weight gradient:
// the same products with a one-hot left operand, done as copies and as sums over sorted tokens.
//
// Backward: dW[v] = scale * sum_{t: id_t = v} dy[t]. Atomics would add in an order that changes from run to run,
// so the tokens are sorted first (stable, by token number) and every row is summed in the order of t:
//   1. the tokens that occur are marked in a bit map;
//   2. one CTA per tile of 16384 tokens sorts the tile in shared memory (radix, up to 9 bits a pass; the items
//      wait in registers between passes, so one copy of the keys is enough), while the other SMs clear the
//      rows of the tokens that do not occur: most of the bytes, and nothing they need from the sort;
//   3. the sorted tokens are cut into chunks of 32 (8 or 16 when they are few), whatever runs of equal tokens they
//      hold: one warp per chunk and 32 vectors of columns. A run inside a chunk goes straight to the table, what
//      crosses a chunk's border to the workspace, so the rows of a token that makes up a tenth of the text are read by as
//      many warps as any others;
//   4. the parts of the runs that cross are added in order, a run's by one warp for each 128 columns (40000 tokens into
//      60000 x 1024: 162 us, 288 when half of them are one token).
// Tiles after the first add to the rows the earlier ones wrote, in launch order: the same bits every time.
#include "nzb_internal.h"
#include "nzb_elem.cuh"

namespace nzb {

constexpr int kSortTile = 16384;
constexpr int kSortThreads = 1024;
constexpr int kSortItems = kSortTile / kSortThreads;
constexpr int kSortMaxBins = 512;
// The rows of the other tokens are cleared beside the sums, not beside the sort, when the sort is short or the table
// small: two launches less (1000 tokens into 30000 x 512: 25 us instead of 45).
constexpr int64_t kFewTokens = 2048, kSmallTable = 8 << 20;  // elements
// Sorted tokens per warp of the sums: few tokens leave SMs idle, and shorter chunks are done sooner, until the joins of long
// runs outweigh that (64 tokens into 14651 x 185: 23.8 us by 32, 16.3 by 16, 15.1 by 8; 1500 into 14652 x 184: 20.5, 17.1, 17.8).
inline int chunk_of(const nzb_embedding_desc* d) { return d->tokens <= 256 ? 8 : d->tokens <= kFewTokens ? 16 : 32; }
inline bool clear_beside_sums(const nzb_embedding_desc* d) { return d->tokens <= kFewTokens || d->vocab * d->dim <= kSmallTable; }
constexpr int kEmbeddingFly = 4;                            // blocks in flight per thread, forward

// What the sort leaves for the sums, per tile.
struct SortTile {
    int32_t count, pad[3];       // tokens that take part
    uint32_t key[kSortTile];     // their numbers, sorted
    int32_t order[kSortTile];    // their positions within the tile
};

struct SortSmem {
    uint32_t key[kSortTile];
    uint32_t hist[32][kSortMaxBins];
    uint32_t bin_base[kSortMaxBins];
    uint16_t pos[kSortTile];
    int32_t scan[32];
};

__device__ __forceinline__ int32_t warp_inclusive_sum(int32_t v, int lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int32_t u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    return v;
}
template <typename Index>
__device__ __forceinline__ uint32_t sort_key(Index index, int64_t vocab, int64_t padding) {
    const int64_t v = static_cast<int64_t>(index);
    return v >= 0 && v < vocab && v != padding ? static_cast<uint32_t>(v) : static_cast<uint32_t>(vocab);
}

template <typename Index>
__global__ void __launch_bounds__(256)
embedding_mark_kernel(const Index* __restrict__ index, int64_t tokens, int64_t vocab, int64_t padding, uint32_t* __restrict__ present) {
    const int64_t t = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    kernel_allow_next();
    if (t >= tokens) return;
    const uint32_t v = sort_key(index[t], vocab, padding);
    if (v != vocab) atomicOr(present + (v >> 5), 1u << (v & 31));
}

// Clears the rows that `present` does not name: a warp per row.
template <class Present>
__device__ __forceinline__ void clear_rows(Present present, float* dtable, int64_t vocab, int64_t dim, int64_t ld_table,
                                           int64_t warp, int64_t warps, int lane) {
    const uint4 zero = make_uint4(0, 0, 0, 0);
    for (int64_t v = warp; v < vocab; v += warps) {
        if (present(v)) continue;
        float* row = dtable + v * ld_table;
        const int lead = row_lead(row);
        for (int64_t c = lane * 4 - lead; c < dim; c += 128) store_block(row, c, dim, zero);
    }
}

// What an earlier kernel of a programmatic launch writes (present, the tiles, the parts) is not `restrict`: such a pointer's
// loads count as independent of everything else and could move before the wait.
template <typename Index>
__global__ void __launch_bounds__(kSortThreads, 1)
embedding_sort_kernel(const Index* __restrict__ index, int64_t tokens, int64_t vocab, int64_t padding, int digit_bits,
                      int passes, int tiles, SortTile* __restrict__ out_tiles, const uint32_t* present,
                      float* __restrict__ dtable, int64_t dim, int64_t ld_table) {
    extern __shared__ uint4 smem_sort[];
    SortSmem& s = *reinterpret_cast<SortSmem*>(smem_sort);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    kernel_allow_next();
    if (blockIdx.x >= tiles) {
        kernel_wait_previous();
        clear_rows([&](int64_t v) { return present[v >> 5] >> (v & 31) & 1; }, dtable, vocab, dim, ld_table,
                   static_cast<int64_t>(blockIdx.x - tiles) * 32 + warp, static_cast<int64_t>(gridDim.x - tiles) * 32, lane);
        return;
    }
    const int64_t t0 = static_cast<int64_t>(blockIdx.x) * kSortTile;
    const int count = static_cast<int>(min(static_cast<int64_t>(kSortTile), tokens - t0));
    SortTile& out = out_tiles[blockIdx.x];
    const uint32_t none = static_cast<uint32_t>(vocab);  // sorts behind every token
    const int rounds = max(1, (count + kSortThreads - 1) / kSortThreads);  // items of a thread: few tokens are soon sorted

    uint32_t k[kSortItems];
    uint16_t p[kSortItems];
#pragma unroll
    for (int i = 0; i < kSortItems; i++) {
        if (i >= rounds) break;
        const int at = warp * (rounds * 32) + i * 32 + lane;
        k[i] = at < count ? sort_key(index[t0 + at], vocab, padding) : none;
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
            if (i >= rounds) break;
            const uint32_t d = (k[i] >> shift) & mask;
            // lanes with the same digit: a ballot per bit (a match instruction takes a turn per different value,
            // which made the pass over the low bits 15 us instead of 4)
            uint32_t peers = 0xffffffffu;
            for (int bit = 0; bit < digit_bits; bit++) {
                const uint32_t set = __ballot_sync(0xffffffffu, d >> bit & 1);
                peers &= d >> bit & 1 ? set : ~set;
            }
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
            if (i >= rounds) break;
            const uint32_t d = (k[i] >> shift) & mask;
            const uint32_t to = s.bin_base[d] + s.hist[warp][d] + rank[i];
            s.key[to] = k[i];
            s.pos[to] = p[i];
        }
        __syncthreads();
        if (pass + 1 < passes) {
#pragma unroll
            for (int i = 0; i < kSortItems; i++) {
                if (i >= rounds) break;
                const int at = warp * (rounds * 32) + i * 32 + lane;
                k[i] = s.key[at];
                p[i] = s.pos[at];
            }
            __syncthreads();
        }
    }
    const int sorted = rounds * kSortThreads;
    for (int i = tid; i < sorted; i += kSortThreads) {
        out.key[i] = s.key[i];
        out.order[i] = s.pos[i];
        if (s.key[i] == none ? i == 0 || s.key[i - 1] != none : i == sorted - 1) out.count = s.key[i] == none ? i : sorted;
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
__global__ void __launch_bounds__(256, ALIGNED ? 4 : 2)
embedding_sum_kernel(const T* __restrict__ dy, const SortTile* tile, float* __restrict__ dtable,
                     float* __restrict__ partial, int64_t vocab, int64_t dim, int64_t ld_table, int64_t ld_y, float scale, int add,
                     int vec_out, unsigned sum_ctas, int chunk_len) {
    constexpr int VEC = Elem<T>::VEC, FLY = 8;  // FLY: rows of dy in flight
    const int lane = threadIdx.x & 31;
    kernel_wait_previous();
    kernel_allow_next();
    if (blockIdx.x >= sum_ctas) {
        // few tokens: the rows of the others are cleared here, found by halving among the sorted ones
        const int count = tile->count;
        const auto present = [&](int64_t v) {
            int lo = 0, hi = count;
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (tile->key[mid] < v) lo = mid + 1;
                else hi = mid;
            }
            return lo < count && tile->key[lo] == v;
        };
        clear_rows(present, dtable, vocab, dim, ld_table, static_cast<int64_t>(blockIdx.x - sum_ctas) * 8 + (threadIdx.x >> 5),
                   static_cast<int64_t>(gridDim.x - sum_ctas) * 8, lane);
        return;
    }
    const int64_t item = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
    const int64_t blocks = (dim + 32 * VEC - 1) / (32 * VEC);  // column blocks of a row
    const int64_t chunk = item / blocks, c0 = (item - chunk * blocks) * 32 * VEC;
    const int count = tile->count, i0 = static_cast<int>(chunk) * chunk_len;
    if (i0 >= count) return;
    const int i1 = min(i0 + chunk_len, count);
    const uint32_t none = 0xffffffffu;
    const uint32_t my_key = i0 + lane < i1 ? tile->key[i0 + lane] : none;
    const int32_t my_row = i0 + lane < i1 ? tile->order[i0 + lane] : 0;
    const uint32_t key_before = i0 > 0 ? tile->key[i0 - 1] : none, key_after = i1 < count ? tile->key[i1] : none;
    const int64_t c = ALIGNED ? c0 + lane * VEC : c0 + lane;
    float acc[VEC];
#pragma unroll
    for (int j = 0; j < VEC; j++) acc[j] = 0.f;
    for (int g = 0; g < i1 - i0; g += FLY) {
        uint4 u[FLY];
        T e[FLY][ALIGNED ? 1 : VEC];
#pragma unroll
        for (int f = 0; f < FLY; f++) {
            const T* row = dy + static_cast<int64_t>(__shfl_sync(0xffffffffu, my_row, g + f)) * ld_y;
            u[f] = make_uint4(0, 0, 0, 0);
            if (g + f < i1 - i0) {
                if (ALIGNED) {
                    if (c < dim) u[f] = load_block(row, c, dim);
                } else {
#pragma unroll
                    for (int j = 0; j < VEC; j++) e[f][ALIGNED ? 0 : j] = c + j * 32 < dim ? row[c + j * 32] : Elem<T>::from(0.f);
                }
            }
        }
#pragma unroll
        for (int f = 0; f < FLY; f++) {
            const int i = g + f;
            if (i >= i1 - i0) break;
            float v[VEC];
            if (ALIGNED) {
                Elem<T>::unpack(u[f], v);
            } else {
#pragma unroll
                for (int j = 0; j < VEC; j++) v[j] = Elem<T>::to(e[f][ALIGNED ? 0 : j]);
            }
#pragma unroll
            for (int j = 0; j < VEC; j++) acc[j] += v[j];
            const uint32_t key = __shfl_sync(0xffffffffu, my_key, i);
            const bool last = i + 1 == i1 - i0;
            const uint32_t next = last ? key_after : __shfl_sync(0xffffffffu, my_key, i + 1);
            if (next == key && !last) continue;
            // the run ends here, or goes on in the next chunk
            const uint32_t first_key = __shfl_sync(0xffffffffu, my_key, 0);
            const bool from_before = key == first_key && key == key_before;
            const bool whole = !from_before && next != key;
            float* to = whole ? dtable + static_cast<int64_t>(key) * ld_table : partial + (2 * chunk + (from_before ? 0 : 1)) * dim;
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
#pragma unroll
            for (int j = 0; j < VEC; j++) acc[j] = 0.f;
        }
    }
}

// Runs over more than one chunk: the warp of the chunk such a run starts in adds its parts, 32 columns x 4.
__global__ void __launch_bounds__(256)
embedding_join_kernel(const SortTile* tile, const float* partial, float* __restrict__ dtable,
                      int64_t dim, int64_t ld_table, float scale, int add, int chunk_len) {
    kernel_wait_previous();
    kernel_allow_next();
    const int lane = threadIdx.x & 31;
    const int64_t item = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
    const int64_t blocks = (dim + 127) / 128;
    const int64_t chunk = item / blocks;
    const int count = tile->count, i0 = static_cast<int>(chunk) * chunk_len, i1 = i0 + chunk_len;
    if (i1 >= count) return;
    const uint32_t key = tile->key[i1 - 1];
    if (tile->key[i1] != key || (i0 > 0 && tile->key[i0 - 1] == key)) return;
    // parts in the chunks behind: one, and one more for every border the run crosses
    int parts = 1;
    for (int i = i1 + chunk_len;; i += 32 * chunk_len) {
        const int at = i + lane * chunk_len;
        const uint32_t ends = __ballot_sync(0xffffffffu, at >= count || tile->key[at] != key);
        parts += ends ? __ffs(ends) - 1 : 32;
        if (ends) break;
    }
    const int64_t c = (item - chunk * blocks) * 128 + lane;
    float acc[4];
#pragma unroll
    for (int j = 0; j < 4; j++) acc[j] = c + j * 32 < dim ? partial[(2 * chunk + 1) * dim + c + j * 32] : 0.f;
#pragma unroll 4
    for (int k = 1; k <= parts; k++)
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (c + j * 32 < dim) acc[j] += partial[2 * (chunk + k) * dim + c + j * 32];
    float* to = dtable + static_cast<int64_t>(key) * ld_table + c;
#pragma unroll
    for (int j = 0; j < 4; j++)
        if (c + j * 32 < dim) to[j * 32] = add ? to[j * 32] + scale * acc[j] : scale * acc[j];
}

// An item is one 16-byte block of y, or one element where a row of the table or of y does not start on 16 bytes. A
// thread takes FLY of them a CTA's width apart, all their loads in flight before the first store.
template <typename Tab, typename Out, typename Index, bool ALIGNED, int FLY>
__global__ void __launch_bounds__(256)
embedding_kernel(const Tab* __restrict__ table, const Index* __restrict__ index, Out* __restrict__ y, int64_t tokens,
                 int64_t vocab, int64_t dim, int64_t ld_table, int64_t ld_y, float scale) {
    constexpr int VEC = ALIGNED ? Elem<Out>::VEC : 1, TV = ALIGNED ? Elem<Tab>::VEC : 1;
    const uint32_t per_row = static_cast<uint32_t>((dim + VEC - 1) / VEC);
    const int64_t item = static_cast<int64_t>(blockIdx.x) * (256 * FLY) + threadIdx.x;
    int64_t t = item >> 32 ? item / per_row : static_cast<uint32_t>(item) / per_row;
    uint32_t b = static_cast<uint32_t>(item - t * per_row);
    const uint32_t rows_on = 256 / per_row, blocks_on = 256 - rows_on * per_row;
    uint4 u[FLY][VEC / TV];
    Tab e[FLY];
    Out* to[FLY];
    int64_t col[FLY];
    bool inside[FLY];
#pragma unroll
    for (int f = 0; f < FLY; f++) {
        col[f] = static_cast<int64_t>(b) * VEC;
        to[f] = nullptr;
        inside[f] = false;
        if (t < tokens) {
            to[f] = y + t * ld_y;
            const int64_t v = static_cast<int64_t>(index[t]);
            inside[f] = v >= 0 && v < vocab;
            const Tab* from = table + (inside[f] ? v : 0) * ld_table;
            if (inside[f]) {
                if (ALIGNED) {
#pragma unroll
                    for (int h = 0; h < VEC / TV; h++) u[f][h] = load_block(from, col[f] + h * TV, dim);
                } else {
                    e[f] = from[b];
                }
            }
        }
        t += rows_on;
        b += blocks_on;
        if (b >= per_row) {
            b -= per_row;
            t++;
        }
    }
#pragma unroll
    for (int f = 0; f < FLY; f++) {
        if (!to[f]) continue;
        if (ALIGNED) {
            float v[Elem<Out>::VEC];
#pragma unroll
            for (int i = 0; i < Elem<Out>::VEC; i++) v[i] = 0.f;
            if (inside[f]) {
#pragma unroll
                for (int h = 0; h < VEC / TV; h++) {
                    float part[Elem<Tab>::VEC];
                    Elem<Tab>::unpack(u[f][h], part);
#pragma unroll
                    for (int i = 0; i < TV; i++) v[h * TV + i] = part[i] * scale;
                }
            }
            store_block(to[f], col[f], dim, Elem<Out>::pack(v));
        } else {
            to[f][col[f]] = Elem<Out>::from(inside[f] ? Elem<Tab>::to(e[f]) * scale : 0.f);
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
    const int64_t most = d->tokens < kSortTile ? d->tokens : kSortTile;
    pl.partial_bytes = (size_t)round_up((most + chunk_of(d) - 1) / chunk_of(d) * 2 * d->dim * 4, 256);  // two borders a chunk
    return pl;
}

template <typename Tab, typename Out, typename Index>
static int launch_embedding(const nzb_embedding_desc* d, const void* table, const void* index, void* y, int sm_count,
                            cudaStream_t s) {
    const bool aligned = aligned_to(table, 16) && aligned_to(y, 16) && d->ld_table * (int64_t)sizeof(Tab) % 16 == 0 &&
                         d->ld_y * (int64_t)sizeof(Out) % 16 == 0;
    const int64_t items = d->tokens * (aligned ? (d->dim + Elem<Out>::VEC - 1) / Elem<Out>::VEC : d->dim);
    // few blocks: a thread for each, so that more SMs take part (32 rows of 4 KB: 2.2 us instead of 2.8)
    const int fly = items <= (int64_t)sm_count * 2048 ? 1 : kEmbeddingFly;
    const int64_t ctas = (items + 256 * fly - 1) / (256 * fly);
    if (ctas > INT32_MAX) return fail(NZB_ERR_UNSUPPORTED, "more than 2^31 CTAs of rows");
    const Tab* tp = static_cast<const Tab*>(table);
    const Index* ip = static_cast<const Index*>(index);
    Out* yp = static_cast<Out*>(y);
    const auto kernel = aligned ? (fly == 1 ? embedding_kernel<Tab, Out, Index, true, 1> : embedding_kernel<Tab, Out, Index, true, kEmbeddingFly>)
                                : (fly == 1 ? embedding_kernel<Tab, Out, Index, false, 1> : embedding_kernel<Tab, Out, Index, false, kEmbeddingFly>);
    kernel<<<(unsigned)ctas, 256, 0, s>>>(tp, ip, yp, d->tokens, d->vocab, d->dim, d->ld_table, d->ld_y, d->scale);
    NZB_CUDA_TRY(cudaGetLastError());
    return NZB_OK;
}

template <typename Index>
static int launch_sort(const nzb_embedding_desc* d, const void* index, const EmbeddingPlan& pl, SortTile* tiles,
                       uint32_t* present, float* dtable, int sm_count, cudaStream_t s) {
    static std::atomic<uint64_t> smem_set{0};
    int rc = ensure_dynamic_smem(smem_set, reinterpret_cast<const void*>(embedding_sort_kernel<Index>), sizeof(SortSmem));
    if (rc != NZB_OK) return rc;
    int bits = 1;
    while (d->vocab >> bits) bits++;  // vocab itself stands for "no token"
    const int passes = (bits + 8) / 9, digit = (bits + passes - 1) / passes;
    const Index* ip = static_cast<const Index*>(index);
    const auto sort = embedding_sort_kernel<Index>;
    if (d->overwrite && !clear_beside_sums(d)) {
        const int64_t first = d->tokens < kSortTile ? d->tokens : kSortTile;
        NZB_CUDA_TRY(cudaMemsetAsync(present, 0, pl.present_bytes, s));
        embedding_mark_kernel<Index><<<(unsigned)((first + 255) / 256), 256, 0, s>>>(ip, first, d->vocab, d->padding_index, present);
        // the sorting CTAs, which need not wait for the marks, fill an SM each; the others share the rows to clear
        const unsigned grid = (unsigned)(pl.tiles + sm_count - (pl.tiles < sm_count / 2 ? pl.tiles : 0));
        NZB_CUDA_TRY(launch_programmatic(sort, grid, kSortThreads, sizeof(SortSmem), s, ip, d->tokens, d->vocab, d->padding_index, digit,
                                         passes, (int)pl.tiles, tiles, present, dtable, d->dim, d->ld_table));
    } else {
        sort<<<(unsigned)pl.tiles, kSortThreads, sizeof(SortSmem), s>>>(ip, d->tokens, d->vocab, d->padding_index, digit, passes,
                                                                       (int)pl.tiles, tiles, present, dtable, d->dim, d->ld_table);
    }
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
    if (!aligned_to(table, dtype_size(d->table_dtype)) || !aligned_to(y, dtype_size(d->dtype)) || !aligned_to(index, index_size(d->index_type)))
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
    if (!aligned_to(dy, dtype_size(d->dtype)) || !aligned_to(dtable, 4) || !aligned_to(index, index_size(d->index_type)))
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
    rc = d->index_type == NZB_I64 ? launch_sort<int64_t>(d, index, pl, tiles, present, dtable, ds->sm_count, s)
                                  : launch_sort<int32_t>(d, index, pl, tiles, present, dtable, ds->sm_count, s);
    if (rc != NZB_OK) return rc;
    const int vec_out = aligned_to(dtable, 16) && d->ld_table % 4 == 0;
    const int chunk = chunk_of(d);
    for (int64_t t = 0; t < pl.tiles; t++) {
        const int add = t > 0 || !d->overwrite;
        const int64_t n = d->tokens - t * kSortTile < kSortTile ? d->tokens - t * kSortTile : kSortTile;
        const int64_t chunks = (n + chunk - 1) / chunk;
        const bool clear = t == 0 && d->overwrite && clear_beside_sums(d);
        NZB_DISPATCH_DTYPE(d->dtype, T, {
            const T* from = static_cast<const T*>(dy) + t * kSortTile * d->ld_y;
            const int64_t warps = chunks * ((d->dim + 32 * Elem<T>::VEC - 1) / (32 * Elem<T>::VEC));
            const unsigned sum_ctas = (unsigned)((warps + 7) / 8);
            int64_t clear_ctas = clear ? (d->vocab + 7) / 8 : 0;
            if (clear_ctas > (int64_t)ds->sm_count * 8) clear_ctas = (int64_t)ds->sm_count * 8;
            const bool rows_aligned = aligned_to(dy, 16) && d->ld_y * (int64_t)sizeof(T) % 16 == 0;
            const auto kernel = rows_aligned ? embedding_sum_kernel<T, true> : embedding_sum_kernel<T, false>;
            if (sum_ctas + clear_ctas)
                NZB_CUDA_TRY(launch_programmatic(kernel, sum_ctas + (unsigned)clear_ctas, 256, 0, s, from, tiles + t, dtable, partial, d->vocab, d->dim,
                                                 d->ld_table, d->ld_y, d->scale, add, vec_out, sum_ctas, chunk));
        });
        if (chunks > 1)
            NZB_CUDA_TRY(launch_programmatic(embedding_join_kernel, (unsigned)((chunks * ((d->dim + 127) / 128) + 7) / 8), 256, 0, s, tiles + t, partial,
                                             dtable, d->dim, d->ld_table, d->scale, add, chunk));
    }
    return NZB_OK;
}

}  // extern "C"
