// Embedding lookup with scaling, and the gradient of its table by sorted ids.
//
//   forward   out[n, :] = scale * table[ids[n], :]          (an id outside [0, V): a row of zeros)
//   backward  gtable[v, :] = scale * sum over {n : ids[n] = v} of gout[n, :]
//
// Both are bound by memory: N D values written (forward), N D read and V D written (backward).
//
// The gradient is a sum over rows that share an id.  A stable radix sort by id brings them together: eight bits per pass, as
// many passes as V has bytes (one for the 98 species), and one block per 2048 rows whose digits' places follow from all blocks'
// counts (those of the first pass from a kernel that also clears the gradient, those of a later one from the pass before).  Then a
// warp takes 32 neighbours of the sorted order, reads their rows sixteen at a time and adds them in the order of the rows in the
// batch; a run of one id that stays inside those 32 is written at once, one that crosses a border leaves its partial sums, which a
// second kernel adds in their order.  No float atomics: the same bits every time, and no row of the table is touched by two warps.
// All sums are float32, scaled and rounded once.
#include <algorithm>

#include "common.cuh"
#include "values.cuh"

namespace cf {
namespace {

constexpr int SORT_THREADS = 512, SORT_WARPS = SORT_THREADS / 32, SORT_ROUNDS = 4, SORT_TILE = SORT_THREADS * SORT_ROUNDS;
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

// A strided table that fits a block's shared memory (the transposed weight of a Linear over the species): read once per block, along
// its columns, and laid out by rows; 29 -> 14 us for 133,120 rows of 128 floats against gathering every value from its own sector.
constexpr int STAGED_BYTES = 96 * 1024;
template <class T, int VEC>
__global__ void __launch_bounds__(512) embed_staged_kernel(const EmbedArgs p, int lanes, int vectors, int ld)
{
    extern __shared__ __align__(16) unsigned char staged[];
    T *rows = reinterpret_cast<T *>(staged);
    const T *table = static_cast<const T *>(p.table);
    const int V = (int)p.V, D = (int)p.D;
    for (int i = threadIdx.x; i < V * D; i += 512) {
        const int d = i / V, v = i - d * V;
        rows[v * ld + d] = table[v * p.row_stride + d * p.col_stride];
    }
    __syncthreads();
    constexpr int ROWS = 8;
    const int lane = threadIdx.x & 31, per_warp = 32 / lanes, part = lane / lanes;
    const long long step = (long long)gridDim.x * 16 * ROWS * per_warp;
    T *out = static_cast<T *>(p.out);
    for (long long first = ((long long)blockIdx.x * 16 + (threadIdx.x >> 5)) * (ROWS * per_warp) + part; first - part < p.N; first += step) {
        long long id[ROWS];
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            const long long n = first + i * per_warp;
            id[i] = n < p.N ? p.ids[n] : -1;
        }
        for (int c = lane % lanes; c < vectors; c += lanes) {
#pragma unroll
            for (int i = 0; i < ROWS; ++i) {
                const long long n = first + i * per_warp;
                float v[VEC];
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[e] = 0.f;
                if (id[i] >= 0 && id[i] < V) {
                    load_values<T, VEC>(rows + (int)id[i] * ld + c * VEC, v);
#pragma unroll
                    for (int e = 0; e < VEC; ++e) v[e] *= p.scale;
                }
                if (n < p.N) store_values<T, VEC>(out + n * p.D + c * VEC, v);
            }
        }
    }
}

template <class T, int VEC>
int launch_staged(const EmbedArgs &p, cudaStream_t s)
{
    static thread_local bool configured[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (!configured[dev & 63]) {
        if (cudaFuncSetAttribute(embed_staged_kernel<T, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize, STAGED_BYTES) != cudaSuccess) {
            cudaGetLastError();
            return fail(CF_ERR_CUDA, "cf_embed_fwd: %d bytes of shared memory not available", STAGED_BYTES);
        }
        configured[dev & 63] = true;
    }
    const int vectors = (int)p.D / VEC, ld = (int)p.D + VEC;  // (a vector more: rows start in different banks)
    int lanes = 1;
    while (lanes < 32 && lanes < vectors) lanes *= 2;
    const size_t bytes = (size_t)p.V * ld * sizeof(T);
    const long long per_block = 16ll * 8 * (32 / lanes), need = (p.N + per_block - 1) / per_block, cap = (long long)sm_count() * 2;
    embed_staged_kernel<T, VEC><<<(unsigned)std::min(need, cap), 512, bytes, s>>>(p, lanes, vectors, ld);
    return launch_status("embed_staged_kernel");
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
int embed_fwd(const EmbedArgs &p, cudaStream_t s)
{
    constexpr int WIDE = 16 / sizeof(T);
    const bool wide_out = p.D % WIDE == 0 && aligned_to(p.out, 16);
    if (p.col_stride == 1 && wide_out && p.row_stride % WIDE == 0 && aligned_to(p.table, 16)) launch_fwd<T, WIDE, false>(p, s);
    else if (wide_out && (p.D + WIDE) * (long long)sizeof(T) <= STAGED_BYTES / p.V && p.N >= 64 * p.V)  // (each block's copy is read back often enough)
        return launch_staged<T, WIDE>(p, s);
    else if (wide_out) launch_fwd<T, WIDE, true>(p, s);
    else launch_fwd<T, 1, true>(p, s);
    return launch_status("embed_fwd_kernel");
}

// ---- sort of the rows by id -------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t key_of(const int64_t *ids, long long n, long long V)
{
    const long long id = ids[n];
    return id >= 0 && id < V ? (uint32_t)id : (uint32_t)V;  // (padded rows sort behind all others)
}

// The first pass' counts, by its first `blocks` blocks; the others clear the gradient, and the counts of the second pass (which its
// predecessor adds to) and the number of runs that cross borders.
struct ClearArgs {
    unsigned char *gtable;
    size_t bytes;
    uint32_t *later;  // counts of the passes behind the first
    size_t later_words;
    uint32_t *runs;
};
__global__ void __launch_bounds__(SORT_THREADS) digit_count_kernel(const int64_t *ids, long long N, long long V, unsigned blocks, uint32_t *counts,
                                                                   const ClearArgs clear)
{
    if (blockIdx.x >= blocks) {
        const size_t at = (size_t)(blockIdx.x - blocks) * SORT_THREADS + threadIdx.x, step = (size_t)(gridDim.x - blocks) * SORT_THREADS;
        const size_t lead = (16 - (reinterpret_cast<uintptr_t>(clear.gtable) & 15)) & 15, head = lead < clear.bytes ? lead : clear.bytes;
        const size_t vectors = (clear.bytes - head) / 16, tail = head + vectors * 16;
        for (size_t i = at; i < vectors; i += step) reinterpret_cast<uint4 *>(clear.gtable + head)[i] = make_uint4(0u, 0u, 0u, 0u);
        for (size_t i = at; i < head; i += step) clear.gtable[i] = 0;
        for (size_t i = tail + at; i < clear.bytes; i += step) clear.gtable[i] = 0;
        for (size_t i = at; i < clear.later_words; i += step) clear.later[i] = 0u;
        if (at == 0) *clear.runs = 0u;
        return;
    }
    __shared__ uint32_t mine[256];
    if (threadIdx.x < 256) mine[threadIdx.x] = 0u;
    __syncthreads();
    const long long base = (long long)blockIdx.x * SORT_TILE;
#pragma unroll
    for (int r = 0; r < SORT_ROUNDS; ++r) {
        const long long n = base + r * SORT_THREADS + threadIdx.x;
        if (n < N) atomicAdd(&mine[key_of(ids, n, V) & 255u], 1u);  // (a count: any order)
    }
    __syncthreads();
    if (threadIdx.x < 256) counts[(size_t)blockIdx.x * 256 + threadIdx.x] = mine[threadIdx.x];
}

// Where there are many blocks of rows: their counts of each digit become those of the blocks before, and the sums over all follow them
// as one more row (each block of the pass reading all blocks' counts itself is quicker up to SCAN_BLOCKS and quadratic).  32 digits per
// block, a share of the rows' blocks per warp.
constexpr unsigned SCAN_BLOCKS = 128;
__global__ void __launch_bounds__(1024) digit_scan_kernel(uint32_t *counts, unsigned blocks)
{
    __shared__ uint32_t part[32][33];
    const unsigned lane = threadIdx.x & 31, warp = threadIdx.x >> 5, d = blockIdx.x * 32 + lane;
    const unsigned lo = (unsigned)((unsigned long long)blocks * warp / 32), hi = (unsigned)((unsigned long long)blocks * (warp + 1) / 32);
    uint32_t sum = 0u;
#pragma unroll 8
    for (unsigned b = lo; b < hi; ++b) sum += counts[(size_t)b * 256 + d];
    part[warp][lane] = sum;
    __syncthreads();
    uint32_t before = 0u;
    for (unsigned w = 0; w < warp; ++w) before += part[w][lane];
#pragma unroll 8
    for (unsigned b = lo; b < hi; ++b) {
        const uint32_t c = counts[(size_t)b * 256 + d];
        counts[(size_t)b * 256 + d] = before;
        before += c;
    }
    if (warp == 31) counts[(size_t)blocks * 256 + d] = before;
}

// One pass: rows to their places by eight bits of their keys, equal digits in their present order; `next`: the counts of the next
// pass' blocks.
__global__ void __launch_bounds__(SORT_THREADS) digit_place_kernel(const int64_t *ids, const uint32_t *keys, const uint32_t *rows, long long N,
                                                                   long long V, int shift, const uint32_t *counts, uint32_t *next, uint32_t *keys_out,
                                                                   uint32_t *rows_out)
{
    __shared__ uint32_t seen[SORT_WARPS][256];  // of a warp's rows so far, then of the warps before
    __shared__ uint32_t place[256], half[2][256], sums[8];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d = threadIdx.x & 255, part = threadIdx.x >> 8;
    const long long base = (long long)blockIdx.x * SORT_TILE + warp * (SORT_ROUNDS * 32) + lane;
    uint32_t key[SORT_ROUNDS], rank[SORT_ROUNDS];
#pragma unroll
    for (int r = 0; r < SORT_ROUNDS; ++r) {
        const long long n = base + r * 32;
        key[r] = n < N ? (keys != nullptr ? keys[n] : key_of(ids, n, V)) : 0u;
    }
    // counts of digit d, of the blocks before this one and of all: half of the blocks each
    uint32_t total = 0u, earlier = 0u;
    if (gridDim.x > SCAN_BLOCKS) {  // (digit_scan_kernel has been there)
        if (!part) {
            total = counts[(size_t)gridDim.x * 256 + d];
            earlier = counts[(size_t)blockIdx.x * 256 + d];
        }
    } else {
        const unsigned mid = (gridDim.x + 1) / 2, lo = part ? mid : 0u, hi = part ? gridDim.x : mid;
#pragma unroll 16
        for (unsigned b = lo; b < hi; ++b) {
            const uint32_t c = counts[(size_t)b * 256 + d];
            total += c;
            earlier += b < blockIdx.x ? c : 0u;
        }
    }
    for (int w = part; w < SORT_WARPS; w += 2) seen[w][d] = 0u;
    __syncthreads();
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
    if (part) { half[0][d] = total; half[1][d] = earlier; }
    __syncthreads();
    uint32_t scan = 0u;
    if (!part) {
        uint32_t own = 0u;
#pragma unroll
        for (int w = 0; w < SORT_WARPS; ++w) {
            const uint32_t t = seen[w][d];
            seen[w][d] = own;
            own += t;
        }
        total += half[0][d];
        earlier += half[1][d];
        scan = total;  // rows of smaller digits: exclusive prefix over the 256 digits
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t t = __shfl_up_sync(FULL, scan, o);
            if (lane >= o) scan += t;
        }
        if (lane == 31) sums[warp] = scan;
    }
    __syncthreads();
    if (!part) {
        uint32_t smaller = scan - total;
#pragma unroll
        for (int w = 0; w < 8; ++w) smaller += w < warp ? sums[w] : 0u;
        place[d] = smaller + earlier;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < SORT_ROUNDS; ++r) {
        const long long n = base + r * 32;
        if (n >= N) break;
        const uint32_t digit = (key[r] >> shift) & 255u, to = place[digit] + seen[warp][digit] + rank[r];
        keys_out[to] = key[r];
        rows_out[to] = rows != nullptr ? rows[n] : (uint32_t)n;
        if (next != nullptr) atomicAdd(&next[(size_t)(to / SORT_TILE) * 256 + ((key[r] >> (shift + 8)) & 255u)], 1u);
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
    uint32_t *runs;                    // how many runs go on behind the chunk that they begin in, then those chunks
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
    constexpr int BATCH = 16;  // rows in flight
    for (int r = 0; r < CHUNK; r += BATCH) {
        if (__shfl_sync(FULL, key, r) == none) break;
        Raw<T, VEC> raw[BATCH];
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const uint32_t k = __shfl_sync(FULL, key, r + i), n = __shfl_sync(FULL, row, r + i);
            raw[i] = Raw<T, VEC>{};
            if (k != none && on) raw[i] = load_raw<T, VEC>(gout + (long long)n * p.ld + col);
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
            float v[VEC];
            expand<T, VEC>(raw[i], v);
#pragma unroll
            for (int e = 0; e < VEC; ++e) acc[e] += v[e];
        }
    }
    // (where the loop ended early, the run before the padded rows is still open; its successor is not of its id)
    finish(run == next);
    if (run == next && run != none && !began_before && lane == 0 && job % p.slabs == 0) p.runs[1 + atomicAdd(p.runs, 1u)] = (uint32_t)chunk;  // (in any order)
}

// Runs that cross borders: a block adds the shares of one run's chunks, its sixteen warps a chunk each in turn.
template <class T, int VEC>
__global__ void __launch_bounds__(512) embed_join_kernel(const SumArgs p)
{
    __shared__ float part[16][32 * VEC];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long chunks = (p.N + CHUNK - 1) / CHUNK;
    const long long jobs = (long long)p.runs[0] * p.slabs;
    for (long long job = blockIdx.x; job < jobs; job += gridDim.x) {
        const long long chunk = p.runs[1 + job / p.slabs];
        const uint32_t id = p.keys[chunk * CHUNK + CHUNK - 1];
        // The last chunk that begins in the run: 32 places tried at a time, neighbours first, then 32 times as far apart each time while
        // all of them are in it, and closer again from the last one that is.
        long long last = chunk + 1, apart = 1;
        bool wider = true;
        while (apart > 0) {
            const long long at = last + apart * lane;
            const int n = __popc(__ballot_sync(FULL, at < chunks && p.keys[at < chunks ? at * CHUNK : 0] == id));  // (sorted: the first n; the one at `last` is)
            last += apart * (n - 1);
            if (n < 32) wider = false;
            apart = wider ? apart * 32 : apart / 32;
        }
        const long long col = ((job % p.slabs) * 32 + lane) * VEC;
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
#pragma unroll 8
            for (long long c = chunk + 1 + warp; c <= last; c += 16) {
                const float *from = p.partial + c * 2 * p.width + col;
#pragma unroll
                for (int e = 0; e < VEC; ++e) acc[e] += from[e];
            }
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < VEC; ++e) part[warp][e * 32 + lane] = acc[e];
        __syncthreads();
        if (warp == 0 && on) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                float t = part[0][e * 32 + lane];
#pragma unroll
                for (int w = 1; w < 16; ++w) t += part[w][e * 32 + lane];
                acc[e] = t;
            }
            store_row<T, VEC>(p, id, col, acc);
        }
    }
}

template <class T, int VEC>
void launch_sums(SumArgs p, cudaStream_t s)
{
    p.slabs = (unsigned)((p.D + 32 * VEC - 1) / (32 * VEC));
    const long long chunks = (p.N + CHUNK - 1) / CHUNK, jobs = chunks * p.slabs;
    embed_sum_kernel<T, VEC><<<(unsigned)((jobs + 7) / 8), 256, 0, s>>>(p);
    if (chunks > 1) embed_join_kernel<T, VEC><<<(unsigned)std::min<long long>((chunks - 1) * p.slabs, 4ll * sm_count()), 512, 0, s>>>(p);
}

template <class T>
void embed_sums(const SumArgs &p, cudaStream_t s)
{
    constexpr int WIDE = 16 / sizeof(T);
    if (p.D % WIDE == 0 && p.ld % WIDE == 0 && aligned_to(p.gout, 16) && aligned_to(p.out, 16)) launch_sums<T, WIDE>(p, s);
    else launch_sums<T, 1>(p, s);
}

struct EmbedWork {
    uint32_t *counts, *keys[2], *rows[2], *runs;
    size_t counts_of;  // words of a pass
    float *partial;
    size_t bytes;
    EmbedWork(void *base, long long N, long long D)
    {
        Carver c{static_cast<char *>(base)};
        counts_of = (size_t)((N + SORT_TILE - 1) / SORT_TILE + 1) * 256;  // (a row for the sums)
        counts = c.take<uint32_t>(4 * counts_of);
        runs = c.take<uint32_t>((size_t)((N + CHUNK - 1) / CHUNK) + 1);
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
    if (type == CF_FLOAT32) return embed_fwd<float>(p, as_stream(stream));
    if (type == CF_BFLOAT16) return embed_fwd<__nv_bfloat16>(p, as_stream(stream));
    return embed_fwd<__half>(p, as_stream(stream));
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
    const size_t bytes = (size_t)V * D * type_size(type);
    if (N == 0) {
        if (cudaMemsetAsync(gtable, 0, bytes, s) != cudaSuccess) return launch_status("cf_embed_bwd: clearing the gradient");
        return CF_OK;
    }
    CF_REQUIRE(gout && ids && workspace, CF_ERR_INVALID, "cf_embed_bwd: null pointer");
    CF_REQUIRE(aligned_to(workspace, 16), CF_ERR_INVALID, "cf_embed_bwd: the workspace does not start on 16 bytes");
    const EmbedWork w(workspace, N, D);
    const unsigned blocks = (unsigned)((N + SORT_TILE - 1) / SORT_TILE);
    const ClearArgs clear{static_cast<unsigned char *>(gtable), bytes, w.counts + w.counts_of, 3 * w.counts_of, w.runs};
    const unsigned clearing = (unsigned)std::max<size_t>(1, std::min<size_t>((bytes / 16 + 3 * w.counts_of) / (SORT_THREADS * 4) + 1, 4 * (size_t)sm_count()));
    digit_count_kernel<<<blocks + clearing, SORT_THREADS, 0, s>>>(ids, N, V, blocks, w.counts, clear);
    const uint32_t *keys = nullptr, *rows = nullptr;
    for (int shift = 0, pass = 0; shift < 32 && (V >> shift) != 0; shift += 8, ++pass) {
        const bool more = shift + 8 < 32 && (V >> (shift + 8)) != 0;
        uint32_t *counts = w.counts + pass * w.counts_of;
        if (blocks > SCAN_BLOCKS) digit_scan_kernel<<<8, 1024, 0, s>>>(counts, blocks);
        digit_place_kernel<<<blocks, SORT_THREADS, 0, s>>>(ids, keys, rows, N, V, shift, counts, more ? counts + w.counts_of : nullptr, w.keys[pass & 1],
                                                           w.rows[pass & 1]);
        keys = w.keys[pass & 1];
        rows = w.rows[pass & 1];
    }
    const SumArgs p{gout, ld, keys, rows, N, V, D, (float)scale, gtable, transposed ? 1 : D, transposed ? V : 1, w.partial, D, w.runs, 1};
    if (type == CF_FLOAT32) embed_sums<float>(p, s);
    else if (type == CF_BFLOAT16) embed_sums<__nv_bfloat16>(p, s);
    else embed_sums<__half>(p, s);
    return launch_status("embed_sum_kernel");
}

}  // extern "C"
