// The gated feed-forward block, forward and backward:
//
//   g = x Wg^T + bg,  u = x Wu^T + bu,  h = act(g) u,  y = h Wd^T + bd
//   dh = gy Wd,  dg = dh u act'(g),  du = dh act(g)
//   gx = dg Wg + du Wu,  gWg = dg^T x,  gWu = du^T x,  gWd = gy^T h,  gbg = sum dg,  gbu = sum du,  gbd = sum gy
//
// 6 N D F operations forward, 12 backward and 4 to compute g and u again (keeping them costs 8 N F bytes each way in float32, which
// take as long as the products up to D of about a thousand).  Forward: one kernel for both projections, the activation and the
// product (tile_gemm.cuh, GLU_FORWARD), one for the projection back.  Backward: one kernel for g, u, dh and all that is element-wise
// (GLU_BACKWARD), one for the three products that give gx, gWg with gWu, and gWd, and one for the biases' sums.
// 16-bit types: h, dg and du are rounded to the type once, as operands of the next product (two values each would double that product:
// 216 of the 391 us backward at 8,192 rows, 1024 x 2816); errors are 1.4 times those of the result's own rounding.  All sums are float32.
// Up to eight rows take no tiles (gated_rows.cuh): the weights are read once, and that is the time.
#include <algorithm>
#include <type_traits>

#include "gated_rows.cuh"
#include "tile_gemm.cuh"

namespace cf {
namespace {

using namespace tile;

// ---- packing: rows of values to planes of pieces with rows on 16 bytes -----------------------------------------------------------
struct PackJob {
    const void *src;
    long long rows, ld;
    int cols;
    Planes to;
    long long groups;  // of eight values, with those that pad a row
    bool transposed;   // rows and cols are those of the planes, the source's the other way round
};
constexpr int PACK_JOBS = 5, COLUMN_SHARES = 512;
struct PackJobs {
    PackJob j[PACK_JOBS];
};

template <class T>
__global__ void __launch_bounds__(256) pack_kernel(const __grid_constant__ PackJobs jobs)
{
    using P = typename Piece<T>::type;
    constexpr int NP = pieces_of<T>;
    const PackJob &job = jobs.j[blockIdx.y];
    grid_launch_dependents();
    grid_dependency_wait();
    const T *src = static_cast<const T *>(job.src);
    P *to = static_cast<P *>(job.to.base);
    const bool wide = ((reinterpret_cast<uintptr_t>(src) & 15) | (job.ld % (16 / (int)sizeof(T)))) == 0;
    const long long per_row = job.to.ld / 8;
    for (long long g = (long long)blockIdx.x * 256 + threadIdx.x; g < job.groups; g += (long long)gridDim.x * 256) {
        // (neighbouring threads read neighbours: along the source's rows)
        const long long row = job.transposed ? g % job.rows : g / per_row;
        const int col = (int)(job.transposed ? g / job.rows : g - row * per_row) * 8, room = job.cols - col;
        float v[8];
        if (job.transposed) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = i < room ? to_float(src[(col + i) * job.ld + row]) : 0.f;
        } else if (wide && room >= 8) {
            constexpr int VEC = 16 / sizeof(T);
#pragma unroll
            for (int i = 0; i < 8; i += VEC) {
                float w[VEC];
                load_values<T, VEC>(src + row * job.ld + col + i, w);
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[i + e] = w[e];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = i < room ? to_float(src[row * job.ld + col + i]) : 0.f;
        }
        uint32_t w[NP][4];
        if constexpr (NP == 3) {
            split_words(v, w);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) w[0][i] = pack_two<P>(v[2 * i], v[2 * i + 1]);
        }
#pragma unroll
        for (int q = 0; q < NP; ++q)
            *reinterpret_cast<uint4 *>(to + q * job.to.plane + row * job.to.ld + col) = make_uint4(w[q][0], w[q][1], w[q][2], w[q][3]);
    }
}

// ---- sums of columns (the biases' gradients) --------------------------------------------------------------------------------------
// Of a matrix of rows in a type (gy) or of float32 sums of 32 rows each (dg and du): a block takes 32 VEC columns of a share of the
// rows, its eight warps rows in turn; the block that brings a column group's last share adds the shares in their order.
struct ColumnJob {
    const void *x;
    long long rows;
    int cols, groups, shares;
    float *partial;       // (shares, cols)
    unsigned *tickets;    // per group
    void *out0, *out1;    // columns [0, cols0), [col1, col1 + cols1)
    int cols0, col1, cols1;
};
struct ColumnJobs {
    ColumnJob j[2];
};
template <class T, class X, int VEC>
__device__ __forceinline__ void sum_columns(const ColumnJob &job, int block)
{
    __shared__ float part[8][32 * VEC];
    __shared__ bool last;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, group = block % job.groups, share = block / job.groups, col = (group * 32 + lane) * VEC;
    const long long lo = job.rows * share / job.shares, hi = job.rows * (share + 1) / job.shares;
    const X *x = static_cast<const X *>(job.x);
    float sum[VEC], low[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) sum[e] = low[e] = 0.f;
    if (col < job.cols) {
#pragma unroll 8
        for (long long n = lo + warp; n < hi; n += 8) {
            float v[VEC];
            load_values<X, VEC>(x + n * job.cols + col, v);
#pragma unroll
            for (int e = 0; e < VEC; ++e) add_compensated(v[e], sum[e], low[e]);
        }
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) part[warp][e * 32 + lane] = fabsf(sum[e]) < INFINITY ? sum[e] + low[e] : sum[e];  // (an infinity loses nothing)
    __syncthreads();
    for (int i = threadIdx.x; i < 32 * VEC; i += 256) {
        const int at = (group * 32 + (i & 31)) * VEC + (i >> 5);
        float t = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) t += part[w][i];
        if (at < job.cols) __stcg(job.partial + (long long)share * job.cols + at, t);
    }
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) last = atomicAdd(job.tickets + group, 1u) + 1u == (unsigned)job.shares;
    __syncthreads();
    if (!last) return;
    __threadfence();
    // (each warp some of the shares, a lane VEC columns as before, then the warps')
#pragma unroll
    for (int e = 0; e < VEC; ++e) sum[e] = 0.f;
    if (col < job.cols) {
#pragma unroll 8
        for (int s = warp; s < job.shares; s += 8) {
            const float *from = job.partial + (long long)s * job.cols + col;
            if constexpr (VEC == 1) {
                sum[0] += __ldcg(from);
            } else {
#pragma unroll
                for (int e = 0; e < VEC; e += 4) {
                    const float4 v = __ldcg(reinterpret_cast<const float4 *>(from + e));
                    sum[e] += v.x; sum[e + 1] += v.y; sum[e + 2] += v.z; sum[e + 3] += v.w;
                }
            }
        }
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) part[warp][lane * VEC + e] = sum[e];
    __syncthreads();
    for (int i = threadIdx.x; i < 32 * VEC; i += 256) {
        const int at = group * 32 * VEC + i;
        float t = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) t += part[w][i];
        if (at >= job.cols) continue;
        if (at < job.cols0) { if (job.out0 != nullptr) static_cast<T *>(job.out0)[at] = from_float<T>(t); }
        else if (at >= job.col1 && at < job.col1 + job.cols1) { if (job.out1 != nullptr) static_cast<T *>(job.out1)[at - job.col1] = from_float<T>(t); }
    }
}
template <class T, int VEC>
__global__ void __launch_bounds__(256) column_sum_kernel(const __grid_constant__ ColumnJobs jobs)
{
    grid_launch_dependents();
    grid_dependency_wait();
    const int first = jobs.j[1].groups * jobs.j[1].shares;  // (the longer shares first)
    if ((int)blockIdx.x < first) sum_columns<T, T, VEC>(jobs.j[1], blockIdx.x);
    else sum_columns<T, float, 4>(jobs.j[0], blockIdx.x - first);
}

// ---- tensor maps ----------------------------------------------------------------------------------------------------------------------
using Encode = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                            const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
Encode encoder()
{
    static const Encode found = [] {
        void *fn = nullptr;
        cudaDriverEntryPointQueryResult state;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &state) != cudaSuccess ||
            state != cudaDriverEntryPointSuccess) {
            cudaGetLastError();
            return static_cast<Encode>(nullptr);
        }
        return reinterpret_cast<Encode>(fn);
    }();
    return found;
}

// Rows of `cols` pieces; what lies beyond them reads as zeros, which is how ragged sizes are done.
template <class T>
int encode(CUtensorMap *map, const Planes &x, long long rows, long long cols, int box_rows)
{
    using P = typename Piece<T>::type;
    const Encode f = encoder();
    CF_REQUIRE(f, CF_ERR_CUDA, "cf_gated_ffn: the driver has no cuTensorMapEncodeTiled");
    const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)pieces_of<T>};
    const cuuint64_t strides[2] = {(cuuint64_t)x.ld * 2, (cuuint64_t)(pieces_of<T> > 1 ? x.plane : x.ld * rows) * 2};
    const cuuint32_t box[3] = {TK, (cuuint32_t)box_rows, 1}, step[3] = {1, 1, 1};
    const CUresult rc = f(map, std::is_same<P, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, x.base, dims, strides,
                          box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    CF_REQUIRE(rc == CUDA_SUCCESS, CF_ERR_CUDA, "cf_gated_ffn: tensor map of %lld x %lld (row stride %lld): error %d", rows, cols, x.ld, (int)rc);
    return CF_OK;
}

struct Operand {
    Planes x;
    long long rows, cols;
};

// ---- launches ----------------------------------------------------------------------------------------------------------------------------
template <class T, int MODE, int TN, bool PAIR>
int launch_tiles(const ParamsOf<MODE> &p, bool chained, cudaStream_t s)
{
    using S = Shape<T, MODE, TN, PAIR>;
    static thread_local int resident[64] = {};  // blocks that the GPU holds at a time (0: not asked yet)
    int dev = 0;
    cudaGetDevice(&dev);
    int &blocks = resident[dev & 63];
    cudaLaunchConfig_t cfg{};
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = S::SMEM;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = PAIR ? 2 : 1; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (blocks == 0) {
        if (cudaFuncSetAttribute(tile_kernel<T, MODE, TN, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM) != cudaSuccess) {
            cudaGetLastError();
            return fail(CF_ERR_CUDA, "cf_gated_ffn: %d bytes of shared memory not available", S::SMEM);
        }
        int clusters = 0;
        cfg.gridDim = dim3(2 * (unsigned)sm_count());
        if (PAIR && (cudaOccupancyMaxActiveClusters(&clusters, tile_kernel<T, MODE, TN, PAIR>, &cfg) != cudaSuccess || clusters < 1)) {
            cudaGetLastError();
            clusters = sm_count() / 2;
        }
        blocks = PAIR ? std::min(2 * clusters, sm_count()) : sm_count();
    }
    long long tiles = 0;
    for (int i = 0; i < p.count; ++i) tiles += p.q[i].tiles;
    cfg.gridDim = dim3((unsigned)std::min<long long>(PAIR ? 2 * tiles : tiles, blocks));
    cfg.numAttrs = chained && chained_launches_enabled() ? 2 : 1;
    if (cudaLaunchKernelEx(&cfg, tile_kernel<T, MODE, TN, PAIR>, p) != cudaSuccess) return launch_status("tile_kernel");
    return launch_status("tile_kernel");
}

// Blocks of a grid-stride kernel over `work` units of one thread each.
unsigned stride_blocks(long long work) { return (unsigned)std::max(1ll, std::min((work + 255) / 256, (long long)sm_count() * 8)); }

int blocks_of(long long K) { return (int)((K + TK - 1) / TK); }

// C (M, N) = sum over parts of A B^T.
struct Linear {
    Operand a[2], b[2];
    bool a_across[2], b_across[2];
    int parts;
    long long K[2];
    long long M;
    int N;
    void *out0, *out1;
    long long rows0, row1, rows1, ld_out;
    bool transposed;
    const void *bias;
    int splits;
};

// How the products of one launch are cut: width of the tiles, one block or a pair of them to a tile, and into how many shares each
// contraction.  Shares are as long as `length` blocks at most, so that the tiles of all products take about as long; the cheapest
// length by the rounds of the launch (blocks of the contraction, and what a tile costs beside them) and by the shares' way through
// memory.  Unit: 256 clocks, the products of 128 x 128 x 64 values of 16 bits.  Measured with each width forced (y; the three gradients):
//   1,984 rows, 128 x 512, float32                pair 256: 25; 31 us   pair 128: 17; 22   single 64: 11; 21
//   133,120 rows, 128 x 512, float32                       163; 669              108; 450            157; 756
//   8,192 rows, 1024 x 2816, bfloat16                       50; 216               84; 355            133; 708
// (single blocks of 128 x 128 were within 5 % of one of them everywhere).  The constants below are fitted to these sizes.
//
// 16-bit types: a share stays in its accumulators from end to end, which lose 1.0e-7 of a sum of one sign with every instruction (the
// gradient of w_down of 131,072 rows, 8,192 instructions, float16: 8.4e-4 too small, 1.7 times half a step of the type).  So no share is longer
// than LONGEST: 1,024 instructions, a fifth of half a step of float16 (1.0e-4 there, whatever the rows).  Backward with it and without:
// 40,000 rows, 1024 x 2048, 1.42 and 1.59 ms; 131,072 rows, 1024 x 2816, 5.7 and 5.7.  (The projections of a tile are not split: 4.2e-4
// at 65,536 features.)
constexpr int LONGEST = 256;
struct Size {
    long long M;
    int N, blocks;
};
struct Cut {
    int tn;
    bool pair;
    int splits[LINEAR_COUNT];
    size_t floats, tickets;  // of all shares, of all warps' parts of split tiles
};
template <class T>
Cut find_cut(const Size *sizes, int count)
{
    // a block of the contraction of a 16-bit type: its products, or what L2 delivers; of float32: six products
    struct Kind { int tn; bool pair; double one, six; };
    constexpr Kind kinds[] = {{256, true, 3.4, 20.0}, {128, true, 3.2, 11.0}, {64, false, 2.2, 7.5}};
    constexpr bool wide = pieces_of<T> > 1;
    const double sms = sm_count();
    int most = 1;
    for (int i = 0; i < count; ++i) most = std::max(most, sizes[i].blocks);
    Cut best{};
    double least = 1e300;
    for (const Kind &k : kinds) {
        const int tm = k.pair ? 2 * TM : TM;
        const double at_once = k.pair ? std::floor(sms / 2) : sms, block = wide ? k.six : k.one;
        for (int length = wide ? most : std::min(most, LONGEST); length >= 1; length = length > 4 ? length * 3 / 4 : length - 1) {
            Cut c{k.tn, k.pair, {}, 0, 0};
            double tiles = 0, work = 0, longest = 0;
            for (int i = 0; i < count; ++i) {
                const Size &z = sizes[i];
                const int splits = (z.blocks + length - 1) / length;
                const double n = (double)((z.M + tm - 1) / tm) * ((z.N + k.tn - 1) / k.tn);
                const double each = std::ceil((double)z.blocks / splits) * block + 4.0 + (splits > 1 ? 1.0 : 0.0);
                c.splits[i] = splits;
                tiles += n * splits;
                work += n * splits * each;
                longest = std::max(longest, each);
                if (splits > 1) {
                    c.floats += (size_t)n * splits * tm * k.tn;
                    c.tickets += (size_t)n * (k.pair ? 2 : 1) * EPILOGUE_WARPS;
                }
            }
            // rounds of tiles of about the same length; 8 bytes a value of a share, at 900 KB a unit
            const double cost = std::max(std::ceil(tiles / at_once) * (work / tiles), longest) + 10.0 + (double)c.floats * 8.0 / 9e5;
            if (cost < least * 0.99) {
                least = cost;
                best = c;
            }
        }
    }
    return best;
}

// The cut of the last sizes asked for is kept, per thread: it costs some microseconds, and a call asks twice (for its workspace's size).
template <class T>
Cut linear_cut(const Size *sizes, int count)
{
    struct Last {
        Size sizes[LINEAR_COUNT];
        int sms = 0;
        Cut cut;
    };
    static thread_local Last last[LINEAR_COUNT];
    Last &l = last[count - 1];
    bool same = l.sms == sm_count();
    for (int i = 0; i < count; ++i) same = same && l.sizes[i].M == sizes[i].M && l.sizes[i].N == sizes[i].N && l.sizes[i].blocks == sizes[i].blocks;
    if (!same) {
        l.cut = find_cut<T>(sizes, count);
        l.sms = sm_count();
        std::copy(sizes, sizes + count, l.sizes);
    }
    return l.cut;
}

template <class T>
int run_linear(const Linear *products, int count, const Cut &cut, float *partial, unsigned *tickets, cudaStream_t s)
{
    if (count == 0) return CF_OK;
    const int tm = cut.pair ? 2 * TM : TM;
    ParamsOf<LINEAR> p{};
    p.count = count;
    p.status = wait_status();
    for (int i = 0; i < count; ++i) {
        const Linear &l = products[i];
        Problem &q = p.q[i];
        for (int part = 0; part < l.parts; ++part) {
            q.a_across[part] = l.a_across[part];
            q.b_across[part] = l.b_across[part];
            int rc = encode<T>(&q.a[part], l.a[part].x, l.a[part].rows, l.a[part].cols, l.a_across[part] ? TK : TM);
            if (rc == CF_OK)
                rc = encode<T>(&q.b[part], l.b[part].x, l.b[part].rows, l.b[part].cols, l.b_across[part] ? TK : cut.pair ? cut.tn / 2 : cut.tn);
            if (rc != CF_OK) return rc;
        }
        q.blocks0 = blocks_of(l.K[0]);
        q.blocks = q.blocks0 + (l.parts > 1 ? blocks_of(l.K[1]) : 0);
        q.M = l.M;
        q.N = l.N;
        q.m_tiles = (int)((l.M + tm - 1) / tm);
        q.n_tiles = (l.N + cut.tn - 1) / cut.tn;
        q.splits = l.splits;
        q.tiles = (long long)q.m_tiles * q.n_tiles * q.splits;
        CF_REQUIRE(q.tiles < (1ll << 31), CF_ERR_RANGE, "cf_gated_ffn: %lld tiles", q.tiles);
        q.out0 = l.out0; q.out1 = l.out1;
        q.rows0 = l.rows0; q.row1 = l.row1; q.rows1 = l.rows1; q.ld_out = l.ld_out;
        q.transposed = l.transposed;
        q.bias = l.bias;
        if (q.splits > 1) {
            q.partial = partial;
            q.tickets = tickets;
            partial += (size_t)q.tiles * tm * cut.tn;
            tickets += (size_t)q.m_tiles * q.n_tiles * (cut.pair ? 2 : 1) * EPILOGUE_WARPS;
        }
    }
    return cut.tn == 256 ? launch_tiles<T, LINEAR, 256, true>(p, true, s) : cut.tn == 128 ? launch_tiles<T, LINEAR, 128, true>(p, true, s) :
                           launch_tiles<T, LINEAR, 64, false>(p, true, s);
}

// ---- plans: where the operands of a call lie ------------------------------------------------------------------------------------------------
long long round_up(long long n, long long to) { return (n + to - 1) / to * to; }

template <class T>
struct Plan {
    static constexpr int NP = pieces_of<T>;
    using P = typename Piece<T>::type;
    const cf_gated_ffn &d;
    long long Fp;
    Operand x, wg, wu, wd, gy, h, dg, du;
    float *partial, *sums = nullptr;  // sums: of the columns of dg and du, 32 rows each
    float *column_shares = nullptr;
    unsigned *tickets;                // of split products, then of column groups
    size_t ticket_words = 0;
    Cut cut;
    size_t bytes;
    PackJobs jobs{};
    int job_count = 0;

    // The matrix itself where TMA can read it (16-bit types on 16 bytes), else its planes in the workspace and the job that makes them.
    Operand place(Carver &c, const void *src, long long rows, long long cols, long long ld, bool transposed = false)
    {
        if (NP == 1 && !transposed && aligned_to(src, 16) && ld % 8 == 0 && ld >= cols && ld < (1ll << 38)) return {{const_cast<void *>(src), ld, 0}, rows, cols};
        const long long to_ld = round_up(cols, 8), plane = rows * to_ld;
        P *to = c.take<P>((size_t)NP * plane);
        jobs.j[job_count++] = {src, rows, ld, (int)cols, {to, to_ld, plane}, rows * (to_ld / 8), transposed};
        return {{to, to_ld, plane}, rows, cols};
    }

    Plan(const cf_gated_ffn &args, const void *gy_src, bool backward, void *base) : d(args), Fp(round_up(args.F, 16))
    {
        Carver c{static_cast<char *>(base)};
        x = place(c, d.x, d.N, d.D, d.ldx);
        wg = place(c, d.w_gate, d.F, d.D, d.D);
        wu = place(c, d.w_up, d.F, d.D, d.D);
        // (the backward's product with it runs across its rows; three pieces, which are packed anyway, are packed transposed)
        wd = backward && NP == 3 ? place(c, d.w_down, d.F, d.D, d.F, true) : place(c, d.w_down, d.D, d.F, d.F);
        if (backward) gy = place(c, gy_src, d.N, d.D, d.D);
        P *hm = c.take<P>((size_t)NP * d.N * Fp);
        h = {{hm, Fp, d.N * Fp}, d.N, d.F};
        if (!backward) {
            const Size y{d.N, (int)d.D, blocks_of(d.F)};
            cut = linear_cut<T>(&y, 1);
        } else {
            P *g = c.take<P>((size_t)NP * d.N * 2 * Fp);
            dg = {{g, 2 * Fp, d.N * 2 * Fp}, d.N, d.F};
            du = {{g ? g + Fp : g, 2 * Fp, d.N * 2 * Fp}, d.N, d.F};
            const int rows = blocks_of(d.N);  // (a call that leaves a gradient out cuts the others the same way)
            const Size every[3] = {{d.N, (int)d.D, 2 * blocks_of(d.F)}, {2 * Fp, (int)d.D, rows}, {d.F, (int)d.D, rows}};
            cut = linear_cut<T>(every, 3);
            sums = c.take<float>((size_t)((d.N + 31) / 32) * 2 * Fp);
            column_shares = c.take<float>((size_t)COLUMN_SHARES * (2 * Fp + d.D));
            ticket_words = (size_t)(2 * Fp + d.D);
        }
        partial = c.take<float>(cut.floats);
        ticket_words += cut.tickets;
        tickets = c.take<unsigned>(ticket_words);
        bytes = c.used;
    }
};

template <class T>
int run_pack(const Plan<T> &plan, cudaStream_t s)
{
    if (plan.job_count == 0) return CF_OK;
    long long most = 0;
    for (int i = 0; i < plan.job_count; ++i) most = std::max(most, plan.jobs.j[i].groups);
    pack_kernel<T><<<dim3(stride_blocks(most), plan.job_count), 256, 0, s>>>(plan.jobs);
    return launch_status("pack_kernel");
}

template <class T>
int run_glu(const Plan<T> &plan, bool backward, bool sums, cudaStream_t s)
{
    const cf_gated_ffn &d = plan.d;
    constexpr bool wide = pieces_of<T> > 1;
    ParamsOf<GLU_FORWARD> p{};
    Problem &q = p.q[0];
    p.count = 1;
    p.clear = plan.tickets;
    p.clear_words = (int)plan.ticket_words;
    // Tiles of pairs (256 x 128; backward in three pieces, whose sums must fit registers, 256 x 64) or of single blocks (128 x 64): the
    // cheaper by rounds times products, single blocks' bound by L2 (16 bits).  Measured (forward; backward), pairs against single blocks:
    // 1,984 rows, 128 x 512, float32 14; 17 us against 9; 17, 133,120 rows 183; 439 against 248; 513, 4,999 rows, 201 x 517, float16
    // 14; 23 against 13; 21, 8,192 rows, 1024 x 2816, bfloat16 91; 173 against 156; 302.
    const int pair_tn = wide && backward ? 64 : 128;
    const double sms = sm_count();
    auto rounds = [&](int tm, int tn, double at_once) { return std::ceil((double)((d.N + tm - 1) / tm) * ((d.F + tn - 1) / tn) / at_once); };
    const double blocks = blocks_of(d.D);
    const bool pair = rounds(256, pair_tn, std::floor(sms / 2)) * pair_tn * (blocks + 2) < rounds(128, 64, sms) * 64 * (blocks + 2) * (wide ? 1.1 : 1.4);
    const int tn = pair ? pair_tn : 64, tm = pair ? 2 * TM : TM;
    const int of_x = backward ? 1 : 0;
    q.blocks0 = blocks_of(d.D);
    q.blocks = backward ? 2 * q.blocks0 : q.blocks0;
    int rc = encode<T>(&q.a[of_x], plan.x.x, d.N, d.D, TM);
    if (rc == CF_OK) rc = encode<T>(&q.b[1], plan.wg.x, d.F, d.D, tn);
    if (rc == CF_OK) rc = encode<T>(&q.b[2], plan.wu.x, d.F, d.D, tn);
    if (backward) {
        if (rc == CF_OK) rc = encode<T>(&q.a[0], plan.gy.x, d.N, d.D, TM);
        if (rc == CF_OK) rc = wide ? encode<T>(&q.b[0], plan.wd.x, d.F, d.D, pair ? tn / 2 : tn) : encode<T>(&q.b[0], plan.wd.x, d.D, d.F, TK);
        q.b_across[0] = !wide;
        p.dg = plan.dg.x;
        p.du = plan.du.x;
        p.sums = sums ? plan.sums : nullptr;
    }
    if (rc != CF_OK) return rc;
    q.m_tiles = (int)((d.N + tm - 1) / tm);
    q.n_tiles = (int)((d.F + tn - 1) / tn);
    q.splits = 1;
    q.tiles = (long long)q.m_tiles * q.n_tiles;
    CF_REQUIRE(q.tiles < (1ll << 31), CF_ERR_RANGE, "cf_gated_ffn: %lld tiles", q.tiles);
    q.M = d.N;
    q.N = (int)d.F;
    p.bias_gate = d.b_gate;
    p.bias_up = d.b_up;
    p.act = d.activation;
    p.h = plan.h.x;
    p.padded = (int)plan.Fp;
    p.status = wait_status();
    const bool chained = plan.job_count > 0;
    if (!pair) return backward ? launch_tiles<T, GLU_BACKWARD, 64, false>(p, chained, s) : launch_tiles<T, GLU_FORWARD, 64, false>(p, chained, s);
    return backward ? launch_tiles<T, GLU_BACKWARD, wide ? 64 : 128, true>(p, chained, s) : launch_tiles<T, GLU_FORWARD, 128, true>(p, chained, s);
}

template <class T>
int forward(const cf_gated_ffn &d, void *y, void *workspace, cudaStream_t s)
{
    if (d.N <= GATED_ROWS) return gated_rows<T>(d, y, static_cast<float *>(workspace), s);
    const Plan<T> plan(d, nullptr, false, workspace);
    int rc = run_pack(plan, s);
    if (rc == CF_OK) rc = run_glu(plan, false, false, s);
    if (rc != CF_OK) return rc;
    Linear l{};
    l.a[0] = plan.h; l.b[0] = plan.wd;
    l.parts = 1;
    l.K[0] = d.F;
    l.M = d.N; l.N = (int)d.D;
    l.out0 = y; l.rows0 = d.N; l.row1 = d.N; l.ld_out = d.D;
    l.bias = d.b_down;
    l.splits = plan.cut.splits[0];
    return run_linear<T>(&l, 1, plan.cut, plan.partial, plan.tickets, s);
}

template <class T>
int run_columns(const Plan<T> &plan, const cf_gated_ffn_grads &g, cudaStream_t s)
{
    const cf_gated_ffn &d = plan.d;
    const int D = (int)d.D, F = (int)d.F, Fp = (int)plan.Fp;
    constexpr int VEC = 16 / sizeof(T);
    const bool wide = D % VEC == 0 && aligned_to(g.gy, 16);
    ColumnJobs jobs{};
    auto place = [&](ColumnJob &j, const void *x, long long rows, int cols, int vec, float *partial, unsigned *tickets) {
        j.x = x; j.rows = rows; j.cols = cols;
        j.groups = (cols + 32 * vec - 1) / (32 * vec);
        // (enough blocks to fill the GPU, of 32 rows at least, few enough for the last one to add up)
        j.shares = (int)std::max(1ll, std::min<long long>({(long long)COLUMN_SHARES, rows / 32, std::max(1ll, 2ll * sm_count() / j.groups)}));
        j.partial = partial; j.tickets = tickets;
    };
    unsigned *tickets = plan.tickets + plan.cut.tickets;
    if (g.b_gate || g.b_up) {
        ColumnJob &j = jobs.j[0];
        place(j, plan.sums, (d.N + 31) / 32, 2 * Fp, 4, plan.column_shares, tickets);
        j.out0 = g.b_gate; j.cols0 = F;
        j.out1 = g.b_up; j.col1 = Fp; j.cols1 = F;
    }
    if (g.b_down) {
        ColumnJob &j = jobs.j[1];
        place(j, g.gy, d.N, D, wide ? VEC : 1, plan.column_shares + (size_t)COLUMN_SHARES * 2 * Fp, tickets + 2 * Fp);
        j.out0 = g.b_down; j.cols0 = D; j.col1 = D;
    }
    const int blocks = jobs.j[0].groups * jobs.j[0].shares + jobs.j[1].groups * jobs.j[1].shares;
    if (blocks == 0) return CF_OK;
    if (wide) launch_chained(column_sum_kernel<T, VEC>, dim3(blocks), dim3(256), 0, s, true, jobs);
    else launch_chained(column_sum_kernel<T, 1>, dim3(blocks), dim3(256), 0, s, true, jobs);
    return launch_status("column_sum_kernel");
}

template <class T>
int backward(const cf_gated_ffn &d, const cf_gated_ffn_grads &g, void *workspace, cudaStream_t s)
{
    const Plan<T> plan(d, g.gy, true, workspace);
    int rc = run_pack(plan, s);
    if (rc == CF_OK) rc = run_glu(plan, true, g.b_gate || g.b_up, s);
    if (rc != CF_OK) return rc;
    const int D = (int)d.D, F = (int)d.F;
    const long long Fp = plan.Fp;
    Linear products[LINEAR_COUNT] = {};
    int count = 0;
    if (g.x) {
        Linear &l = products[count++];
        l.a[0] = plan.dg; l.b[0] = plan.wg;
        l.a[1] = plan.du; l.b[1] = plan.wu;
        l.b_across[0] = l.b_across[1] = true;
        l.parts = 2;
        l.K[0] = l.K[1] = F;
        l.M = d.N; l.N = D;
        l.out0 = g.x; l.rows0 = d.N; l.row1 = d.N; l.ld_out = D;
        l.splits = plan.cut.splits[0];
    }
    if (g.w_gate || g.w_up) {  // one product for both: rows [0, F) and [Fp, Fp + F)
        Linear &l = products[count++];
        l.a[0] = {plan.dg.x, d.N, 2 * Fp}; l.b[0] = plan.x;
        l.a_across[0] = l.b_across[0] = true;
        l.parts = 1;
        l.K[0] = d.N;
        l.M = 2 * Fp; l.N = D;
        l.out0 = g.w_gate; l.rows0 = g.w_gate ? F : 0;
        l.out1 = g.w_up; l.row1 = Fp; l.rows1 = g.w_up ? F : 0;
        l.ld_out = D;
        l.splits = plan.cut.splits[1];
    }
    if (g.w_down) {
        Linear &l = products[count++];
        // h^T gy, stored transposed: F is the larger side as a rule, and tiles are taller than they are wide
        l.a[0] = plan.h; l.b[0] = plan.gy;
        l.a_across[0] = l.b_across[0] = true;
        l.parts = 1;
        l.K[0] = d.N;
        l.M = F; l.N = D;
        l.out0 = g.w_down; l.rows0 = F; l.row1 = F; l.ld_out = F;
        l.transposed = true;
        l.splits = plan.cut.splits[2];
    }
    if ((rc = run_linear<T>(products, count, plan.cut, plan.partial, plan.tickets, s)) != CF_OK) return rc;
    return run_columns(plan, g, s);
}

int check_args(const char *who, const cf_gated_ffn *d)
{
    CF_REQUIRE(d, CF_ERR_INVALID, "%s: null pointer", who);
    CF_REQUIRE(known_type(d->type), CF_ERR_UNSUPPORTED, "%s: type %d is none of CF_FLOAT32, CF_BFLOAT16, CF_FLOAT16", who, d->type);
    CF_REQUIRE(d->activation >= CF_GATE_SILU && d->activation <= CF_GATE_RELU, CF_ERR_UNSUPPORTED, "%s: activation %d", who, d->activation);
    CF_REQUIRE(d->N >= 0 && d->D >= 1 && d->F >= 1 && d->ldx >= 0, CF_ERR_INVALID, "%s: N=%lld D=%lld F=%lld", who, (long long)d->N, (long long)d->D,
               (long long)d->F);
    CF_REQUIRE(d->N <= (1ll << 26) && d->D <= 65536 && d->F <= 262144, CF_ERR_RANGE, "%s: N=%lld D=%lld F=%lld exceed 2^26, 2^16, 2^18", who,
               (long long)d->N, (long long)d->D, (long long)d->F);
    CF_REQUIRE(d->w_gate && d->w_up && d->w_down && (d->N == 0 || d->x), CF_ERR_INVALID, "%s: null pointer", who);
    return CF_OK;
}

template <class T>
size_t workspace_bytes(const cf_gated_ffn &d, const void *gy, bool back)
{
    if (!back && d.N <= GATED_ROWS) return (size_t)d.N * d.F * sizeof(float);
    return Plan<T>(d, gy, back, nullptr).bytes;
}

}  // namespace
}  // namespace cf

using namespace cf;

extern "C" {

int64_t cf_gated_ffn_workspace_bytes(const cf_gated_ffn *args, const void *gy, int backward)
{
    if (check_args("cf_gated_ffn_workspace_bytes", args) != CF_OK || args->N == 0) return 0;
    const bool back = backward != 0;
    if (args->type == CF_FLOAT32) return (int64_t)workspace_bytes<float>(*args, gy, back);
    if (args->type == CF_BFLOAT16) return (int64_t)workspace_bytes<__nv_bfloat16>(*args, gy, back);
    return (int64_t)workspace_bytes<__half>(*args, gy, back);
}

int cf_gated_ffn_fwd(const cf_gated_ffn *args, void *y, void *workspace, void *stream)
{
    int rc = check_args("cf_gated_ffn_fwd", args);
    if (rc != CF_OK || args->N == 0) return rc;
    CF_REQUIRE(y && workspace, CF_ERR_INVALID, "cf_gated_ffn_fwd: null pointer");
    CF_REQUIRE(aligned_to(workspace, 256), CF_ERR_INVALID, "cf_gated_ffn_fwd: the workspace does not start on 256 bytes");
    if ((rc = check_waits("cf_gated_ffn_fwd")) != CF_OK) return rc;
    cudaStream_t s = as_stream(stream);
    if (args->type == CF_FLOAT32) return forward<float>(*args, y, workspace, s);
    if (args->type == CF_BFLOAT16) return forward<__nv_bfloat16>(*args, y, workspace, s);
    return forward<__half>(*args, y, workspace, s);
}

int cf_gated_ffn_bwd(const cf_gated_ffn *args, const cf_gated_ffn_grads *grads, void *workspace, void *stream)
{
    int rc = check_args("cf_gated_ffn_bwd", args);
    if (rc != CF_OK) return rc;
    CF_REQUIRE(grads, CF_ERR_INVALID, "cf_gated_ffn_bwd: null pointer");
    cudaStream_t s = as_stream(stream);
    if (args->N == 0) {  // sums over no rows
        const size_t size = type_size(args->type), D = args->D, F = args->F;
        const std::pair<void *, size_t> empty[] = {{grads->w_gate, F * D}, {grads->w_up, F * D}, {grads->w_down, D * F}, {grads->b_gate, F}, {grads->b_up, F}, {grads->b_down, D}};
        for (const auto &e : empty)
            if (e.first && cudaMemsetAsync(e.first, 0, e.second * size, s) != cudaSuccess) return launch_status("cf_gated_ffn_bwd");
        return CF_OK;
    }
    CF_REQUIRE(grads->gy && workspace, CF_ERR_INVALID, "cf_gated_ffn_bwd: null pointer");
    CF_REQUIRE(aligned_to(workspace, 256), CF_ERR_INVALID, "cf_gated_ffn_bwd: the workspace does not start on 256 bytes");
    if ((rc = check_waits("cf_gated_ffn_bwd")) != CF_OK) return rc;
    if (args->type == CF_FLOAT32) return backward<float>(*args, *grads, workspace, s);
    if (args->type == CF_BFLOAT16) return backward<__nv_bfloat16>(*args, *grads, workspace, s);
    return backward<__half>(*args, *grads, workspace, s);
}

}  // extern "C"
