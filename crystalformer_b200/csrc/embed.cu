// Embedding lookup with scaling, and the gradient of its table by sorted ids.
//
//   forward   out[n, :] = scale * table[ids[n], :]          (an id outside [0, V): a row of zeros)
//   backward  gtable[v, :] = scale * sum over {n : ids[n] = v} of gout[n, :]
//
// Both are bound by memory: N D values written (forward), N D read and V D written (backward).
//
// The gradient is a sum over rows that share an id.  A stable radix sort by id brings them together: eight bits per pass, as
// many passes as V has bytes (one for the 98 species), and one block per 2048 rows whose digits' places follow from all blocks'
// counts.  Then a warp takes 32 neighbours of the sorted order, reads their rows eight at a time and adds them in the order of
// the rows in the batch; a run of one id that stays inside those 32 is written at once, one that crosses a border leaves its
// partial sums, which a second kernel adds in their order.  No atomics: the same bits every time, and no row of the table is
// touched by two warps.  All sums are float32, scaled and rounded once.
#include <algorithm>

#include "common.cuh"
#include "values.cuh"

namespace cf {
namespace {

constexpr int SORT_THREADS = 256, SORT_ROUNDS = 8, SORT_TILE = SORT_THREADS * SORT_ROUNDS;
constexpr int CHUNK = 32;  // neighbours of the sorted order per warp

struct EmbedArgs {
    const void *table;
    long long row_stride, col_stride;
    const int64_t *ids;
    long long N, V, D;
    float scale;
    void *out;
};

// ---- forward ----------------------------------------------------------------------------------------------------------------
// `lanes` (a power of two) neighbours share a row; ROWS rows of a warp's share are in flight at a time.
template <class T, int VEC, bool STRIDED>
__global__ void __launch_bounds__(256) embed_fwd_kernel(const EmbedArgs p, int lanes, long long vectors)
{
    constexpr int ROWS = 4;
    const int lane = threadIdx.x & 31, per_warp = 32 / lanes;
    const long long warp = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const long long first = warp * (ROWS * per_warp) + lane / lanes;
    const T *table = static_cast<const T *>(p.table);
    T *out = static_cast<T *>(p.out);
    long long id[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const long long n = first + (long long)i * per_warp;
        id[i] = n < p.N ? p.ids[n] : -1;
    }
    for (long long c = lane % lanes; c < vectors; c += lanes) {
        float v[ROWS][VEC];
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[i][e] = 0.f;
            if (id[i] >= 0 && id[i] < p.V) {
                const T *at = table + id[i] * p.row_stride + c * VEC * p.col_stride;
                if constexpr (STRIDED) {
#pragma unroll
                    for (int e = 0; e < VEC; ++e) v[i][e] = to_float(at[e * p.col_stride]);
                } else {
                    load_values<T, VEC>(at, v[i]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            const long long n = first + (long long)i * per_warp;
            if (n >= p.N) break;
            if (id[i] >= 0 && id[i] < p.V) {  // (a padded row stays zero whatever the scale)
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[i][e] *= p.scale;
            }
            store_values<T, VEC>(out + n * p.D + c * VEC, v[i]);
        }
    }
}

template <class T, int VEC, bool STRIDED>
void launch_fwd(const EmbedArgs &p, cudaStream_t s)
{
    const long long vectors = p.D / VEC;
    int lanes = 1;
    while (lanes < 32 && lanes < vectors) lanes *= 2;
    const long long per_block = 8ll * 4 * (32 / lanes);
    embed_fwd_kernel<T, VEC, STRIDED><<<(unsigned)((p.N + per_block - 1) / per_block), 256, 0, s>>>(p, lanes, vectors);
}

template <class T>
void embed_fwd(const EmbedArgs &p, cudaStream_t s)
{
    constexpr int WIDE = 16 / sizeof(T);
    const bool wide_out = p.D % WIDE == 0 && aligned_to(p.out, 16);
    if (p.col_stride == 1 && wide_out && p.row_stride % WIDE == 0 && aligned_to(p.table, 16)) launch_fwd<T, WIDE, false>(p, s);
    else if (wide_out) launch_fwd<T, WIDE, true>(p, s);
    else launch_fwd<T, 1, true>(p, s);
}

// ---- sort of the rows by id -------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t key_of(const int64_t *ids, long long n, long long V)
{
    const long long id = ids[n];
    return id >= 0 && id < V ? (uint32_t)id : (uint32_t)V;  // (padded rows sort behind all others)
}

__global__ void __launch_bounds__(SORT_THREADS) digit_count_kernel(const int64_t *ids, const uint32_t *keys, long long N, long long V, int shift,
                                                                   uint32_t *counts)
{
    __shared__ uint32_t mine[256];
    mine[threadIdx.x] = 0u;
    __syncthreads();
    const long long base = (long long)blockIdx.x * SORT_TILE;
#pragma unroll
    for (int r = 0; r < SORT_ROUNDS; ++r) {
        const long long n = base + r * SORT_THREADS + threadIdx.x;
        if (n < N) atomicAdd(&mine[((keys != nullptr ? keys[n] : key_of(ids, n, V)) >> shift) & 255u], 1u);  // (a count: any order)
    }
    __syncthreads();
    counts[(size_t)blockIdx.x * 256 + threadIdx.x] = mine[threadIdx.x];
}

// One pass: rows to their places by eight bits of their keys, equal digits in their present order.
__global__ void __launch_bounds__(SORT_THREADS) digit_place_kernel(const int64_t *ids, const uint32_t *keys, const uint32_t *rows, long long N,
                                                                   long long V, int shift, const uint32_t *counts, uint32_t *keys_out,
                                                                   uint32_t *rows_out)
{
    __shared__ uint32_t seen[8][256];  // of a warp's rows so far, then of the warps before
    __shared__ uint32_t place[256], sums[8];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d = threadIdx.x;
#pragma unroll
    for (int w = 0; w < 8; ++w) seen[w][d] = 0u;
    __syncthreads();
    const long long base = (long long)blockIdx.x * SORT_TILE + warp * (SORT_ROUNDS * 32) + lane;
    uint32_t key[SORT_ROUNDS], rank[SORT_ROUNDS];
#pragma unroll
    for (int r = 0; r < SORT_ROUNDS; ++r) {
        const long long n = base + r * 32;
        key[r] = n < N ? (keys != nullptr ? keys[n] : key_of(ids, n, V)) : 0u;
    }
#pragma unroll
    for (int r = 0; r < SORT_ROUNDS; ++r) {
        const bool on = base + r * 32 < N;
        const uint32_t digit = on ? (key[r] >> shift) & 255u : 256u;
        const uint32_t same = __match_any_sync(FULL, digit);
        const uint32_t before = __popc(same & ((1u << lane) - 1u));
        rank[r] = on ? seen[warp][digit] + before : 0u;
        __syncwarp();
        if (on && before == 0u) seen[warp][digit] += __popc(same);
        __syncwarp();
    }
    __syncthreads();
    uint32_t own = 0u, total = 0u, earlier = 0u;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
        const uint32_t t = seen[w][d];
        seen[w][d] = own;
        own += t;
    }
    if (gridDim.x == 1) {
        total = own;
    } else {
#pragma unroll 8
        for (unsigned b = 0; b < gridDim.x; ++b) {
            const uint32_t c = counts[(size_t)b * 256 + d];
            total += c;
            earlier += b < blockIdx.x ? c : 0u;
        }
    }
    uint32_t scan = total;  // rows of smaller digits: exclusive prefix over the 256 digits
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t t = __shfl_up_sync(FULL, scan, o);
        if (lane >= o) scan += t;
    }
    if (lane == 31) sums[warp] = scan;
    __syncthreads();
    uint32_t smaller = scan - total;
#pragma unroll
    for (int w = 0; w < 8; ++w) smaller += w < warp ? sums[w] : 0u;
    place[d] = smaller + earlier;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < SORT_ROUNDS; ++r) {
        const long long n = base + r * 32;
        if (n >= N) break;
        const uint32_t digit = (key[r] >> shift) & 255u, to = place[digit] + seen[warp][digit] + rank[r];
        keys_out[to] = key[r];
        rows_out[to] = rows != nullptr ? rows[n] : (uint32_t)n;
    }
}

// ---- sums of the sorted rows ---------------------------------------------------------------------------------------------------
struct SumArgs {
    const void *gout;
    long long ld;
    const uint32_t *keys, *rows;
    long long N, V, D;
    float scale;
    void *out;
    long long row_stride, col_stride;  // of out
    float *partial;                    // (chunks, 2, width): of a run that began before the chunk, and of one that goes on behind it
    long long width;
    unsigned slabs;
};

template <class T, int VEC>
__device__ __forceinline__ void store_row(const SumArgs &p, uint32_t id, long long col, const float (&acc)[VEC])
{
    T *to = static_cast<T *>(p.out) + (long long)id * p.row_stride + col * p.col_stride;
    float v[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = acc[e] * p.scale;
    if (p.col_stride == 1) {
        store_values<T, VEC>(to, v);
    } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) to[e * p.col_stride] = from_float<T>(v[e]);
    }
}

template <class T, int VEC>
__global__ void __launch_bounds__(256) embed_sum_kernel(const SumArgs p)
{
    const int lane = threadIdx.x & 31;
    const long long job = (long long)blockIdx.x * 8 + (threadIdx.x >> 5), chunk = job / p.slabs, n0 = chunk * CHUNK;
    if (n0 >= p.N) return;
    const long long col = ((job % p.slabs) * 32 + lane) * VEC;
    const bool on = col < p.D;
    const bool inside = n0 + lane < p.N;
    const uint32_t none = (uint32_t)p.V;
    const uint32_t key = inside ? p.keys[n0 + lane] : none, row = inside ? p.rows[n0 + lane] : 0u;
    const uint32_t prev = n0 > 0 ? p.keys[n0 - 1] : none, next = n0 + CHUNK < p.N ? p.keys[n0 + CHUNK] : none;
    const T *gout = static_cast<const T *>(p.gout);
    float acc[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
    uint32_t run = __shfl_sync(FULL, key, 0);
    bool began_before = run == prev;
    auto finish = [&](bool goes_on) {
        if (run == none || !on) return;
        if (began_before || goes_on) {
            float *to = p.partial + (chunk * 2 + (began_before ? 0 : 1)) * p.width + col;
#pragma unroll
            for (int e = 0; e < VEC; ++e) to[e] = acc[e];
        } else {
            store_row<T, VEC>(p, run, col, acc);
        }
    };
    constexpr int BATCH = 8;  // rows in flight
    for (int r = 0; r < CHUNK; r += BATCH) {
        if (__shfl_sync(FULL, key, r) == none) break;
        float v[BATCH][VEC];
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const uint32_t k = __shfl_sync(FULL, key, r + i), n = __shfl_sync(FULL, row, r + i);
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[i][e] = 0.f;
            if (k != none && on) load_values<T, VEC>(gout + (long long)n * p.ld + col, v[i]);
        }
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const uint32_t k = __shfl_sync(FULL, key, r + i);
            if (k != run) {
                finish(false);
                run = k;
                began_before = false;
#pragma unroll
                for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) acc[e] += v[i][e];
        }
    }
    // (where the loop ended early, the run before the padded rows is still open; its successor is not of its id)
    finish(run == next);
}

// Runs that cross borders: the block of the chunk in which one begins adds the chunks' shares, eight warps a chunk each in turn.
template <class T, int VEC>
__global__ void __launch_bounds__(256) embed_join_kernel(const SumArgs p)
{
    __shared__ float part[8][32 * VEC];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long chunk = blockIdx.x / p.slabs, n0 = chunk * CHUNK;
    if (n0 + CHUNK >= p.N) return;
    const uint32_t id = p.keys[n0 + CHUNK - 1];
    if (id >= (uint32_t)p.V || p.keys[n0 + CHUNK] != id) return;
    if (n0 > 0 && p.keys[n0] == id && p.keys[n0 - 1] == id) return;  // begins in an earlier chunk
    long long lo = n0 + CHUNK, hi = p.N;  // the run's end: keys[lo] == id, keys[hi] is not
    while (hi - lo > 1) {
        const long long mid = (lo + hi) >> 1;
        if (p.keys[mid] == id) lo = mid;
        else hi = mid;
    }
    const long long last = lo / CHUNK, col = ((long long)(blockIdx.x % p.slabs) * 32 + lane) * VEC;
    const bool on = col < p.D;
    float acc[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
    if (on) {
        if (warp == 0) {
            const float *from = p.partial + (chunk * 2 + 1) * p.width + col;
#pragma unroll
            for (int e = 0; e < VEC; ++e) acc[e] = from[e];
        }
#pragma unroll 4
        for (long long c = chunk + 1 + warp; c <= last; c += 8) {
            const float *from = p.partial + c * 2 * p.width + col;
#pragma unroll
            for (int e = 0; e < VEC; ++e) acc[e] += from[e];
        }
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) part[warp][e * 32 + lane] = acc[e];
    __syncthreads();
    if (warp == 0 && on) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            float t = part[0][e * 32 + lane];
#pragma unroll
            for (int w = 1; w < 8; ++w) t += part[w][e * 32 + lane];
            acc[e] = t;
        }
        store_row<T, VEC>(p, id, col, acc);
    }
}

template <class T, int VEC>
void launch_sums(SumArgs p, cudaStream_t s)
{
    p.slabs = (unsigned)((p.D + 32 * VEC - 1) / (32 * VEC));
    const long long chunks = (p.N + CHUNK - 1) / CHUNK, jobs = chunks * p.slabs;
    embed_sum_kernel<T, VEC><<<(unsigned)((jobs + 7) / 8), 256, 0, s>>>(p);
    if (chunks > 1) embed_join_kernel<T, VEC><<<(unsigned)((chunks - 1) * p.slabs), 256, 0, s>>>(p);
}

template <class T>
void embed_sums(const SumArgs &p, cudaStream_t s)
{
    constexpr int WIDE = 16 / sizeof(T);
    if (p.D % WIDE == 0 && p.ld % WIDE == 0 && aligned_to(p.gout, 16) && aligned_to(p.out, 16)) launch_sums<T, WIDE>(p, s);
    else launch_sums<T, 1>(p, s);
}

struct EmbedWork {
    uint32_t *counts, *keys[2], *rows[2];
    float *partial;
    size_t bytes;
    EmbedWork(void *base, long long N, long long D)
    {
        Carver c{static_cast<char *>(base)};
        counts = c.take<uint32_t>((size_t)((N + SORT_TILE - 1) / SORT_TILE) * 256);
        for (int i = 0; i < 2; ++i) { keys[i] = c.take<uint32_t>(N); rows[i] = c.take<uint32_t>(N); }
        partial = c.take<float>((size_t)((N + CHUNK - 1) / CHUNK) * 2 * D);
        bytes = c.used;
    }
};

int check_sizes(const char *who, int type, int64_t N, int64_t V, int64_t D)
{
    CF_REQUIRE(known_type(type), CF_ERR_UNSUPPORTED, "%s: type %d is none of CF_FLOAT32, CF_BFLOAT16, CF_FLOAT16", who, type);
    CF_REQUIRE(N >= 0 && V >= 1 && D >= 1, CF_ERR_INVALID, "%s: N=%lld V=%lld D=%lld", who, (long long)N, (long long)V, (long long)D);
    CF_REQUIRE(N <= CF_EMBED_MAX_ROWS && V <= CF_EMBED_MAX_ROWS && D <= 65536, CF_ERR_RANGE, "%s: N=%lld V=%lld D=%lld exceed 2^30, 2^30, 65536", who,
               (long long)N, (long long)V, (long long)D);
    // one block's share of rows and columns, times the number of blocks that a launch may have
    CF_REQUIRE(N / 32 * ((D + 31) / 32) < (1ll << 31) - 64, CF_ERR_RANGE, "%s: N=%lld rows of D=%lld are more than one launch holds", who, (long long)N,
               (long long)D);
    return CF_OK;
}

}  // namespace
}  // namespace cf

using namespace cf;

extern "C" {

int cf_embed_fwd(const void *table, int64_t row_stride, int64_t col_stride, int type, const int64_t *ids, int64_t N, int64_t V, int64_t D, double scale,
                 void *out, void *stream)
{
    const int rc = check_sizes("cf_embed_fwd", type, N, V, D);
    if (rc != CF_OK) return rc;
    if (N == 0) return CF_OK;
    CF_REQUIRE(table && ids && out, CF_ERR_INVALID, "cf_embed_fwd: null pointer");
    CF_REQUIRE(row_stride >= 0 && col_stride >= 0, CF_ERR_INVALID, "cf_embed_fwd: strides %lld, %lld", (long long)row_stride, (long long)col_stride);
    const EmbedArgs p{table, row_stride, col_stride, ids, N, V, D, (float)scale, out};
    if (type == CF_FLOAT32) embed_fwd<float>(p, as_stream(stream));
    else if (type == CF_BFLOAT16) embed_fwd<__nv_bfloat16>(p, as_stream(stream));
    else embed_fwd<__half>(p, as_stream(stream));
    return launch_status("embed_fwd_kernel");
}

int64_t cf_embed_bwd_workspace_bytes(int64_t N, int64_t D) { return N < 0 || D < 0 ? 0 : (int64_t)EmbedWork(nullptr, N, D).bytes; }

int cf_embed_bwd(const void *gout, int64_t ld, int type, const int64_t *ids, int64_t N, int64_t V, int64_t D, double scale, void *gtable, int transposed,
                 void *workspace, void *stream)
{
    const int rc = check_sizes("cf_embed_bwd", type, N, V, D);
    if (rc != CF_OK) return rc;
    CF_REQUIRE(gtable, CF_ERR_INVALID, "cf_embed_bwd: null pointer");
    CF_REQUIRE(ld >= 0, CF_ERR_INVALID, "cf_embed_bwd: row stride %lld", (long long)ld);
    cudaStream_t s = as_stream(stream);
    if (cudaMemsetAsync(gtable, 0, (size_t)V * D * type_size(type), s) != cudaSuccess) return launch_status("cf_embed_bwd: clearing the gradient");
    if (N == 0) return CF_OK;
    CF_REQUIRE(gout && ids && workspace, CF_ERR_INVALID, "cf_embed_bwd: null pointer");
    CF_REQUIRE(aligned_to(workspace, 16), CF_ERR_INVALID, "cf_embed_bwd: the workspace does not start on 16 bytes");
    const EmbedWork w(workspace, N, D);
    const unsigned blocks = (unsigned)((N + SORT_TILE - 1) / SORT_TILE);
    const uint32_t *keys = nullptr, *rows = nullptr;
    for (int shift = 0, to = 0; shift < 32 && (V >> shift) != 0; shift += 8, to ^= 1) {
        if (blocks > 1) digit_count_kernel<<<blocks, SORT_THREADS, 0, s>>>(ids, keys, N, V, shift, w.counts);
        digit_place_kernel<<<blocks, SORT_THREADS, 0, s>>>(ids, keys, rows, N, V, shift, w.counts, w.keys[to], w.rows[to]);
        keys = w.keys[to];
        rows = w.rows[to];
    }
    const SumArgs p{gout, ld, keys, rows, N, V, D, (float)scale, gtable, transposed ? 1 : D, transposed ? V : 1, w.partial, D, 1};
    if (type == CF_FLOAT32) embed_sums<float>(p, s);
    else if (type == CF_BFLOAT16) embed_sums<__nv_bfloat16>(p, s);
    else embed_sums<__half>(p, s);
    return launch_status("embed_sum_kernel");
}

}  // extern "C"
