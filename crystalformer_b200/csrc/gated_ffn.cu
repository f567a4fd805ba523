// The gated feed-forward block, forward and backward:
//
//   g = x Wg^T + bg,  u = x Wu^T + bu,  h = act(g) u,  y = h Wd^T + bd
//   dh = gy Wd,  dg = dh u act'(g),  du = dh act(g)
//   gx = dg Wg + du Wu,  gWg = dg^T x,  gWu = du^T x,  gWd = gy^T h,  gbg = sum dg,  gbu = sum du,  gbd = sum gy
//
// 6 N D F operations forward, 12 backward and 4 to compute g and u again (keeping them costs 8 N F bytes each way in float32, which
// take as long as the products up to D of about a thousand).  Forward: one kernel for both projections, the activation and the
// product (tile_gemm.cuh, GLU_FORWARD), one for the projection back.  Backward: one kernel for g, u, dh and all that is element-wise
// (GLU_BACKWARD), one for gx, one for both gate weights' gradients, one for gWd, and sums of columns for the biases.
// 16-bit types: h, dg and du are rounded to the type once, as operands of the next product; all sums are float32.
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
constexpr int PACK_JOBS = 5, COLUMN_SHARES = 256;
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
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (NP == 3) {
                uint32_t s[3];
                split_words(v[2 * i], v[2 * i + 1], s);
#pragma unroll
                for (int q = 0; q < 3; ++q) w[q][i] = s[q];
            } else {
                w[0][i] = pack_two<P>(v[2 * i], v[2 * i + 1]);
            }
        }
#pragma unroll
        for (int q = 0; q < NP; ++q)
            *reinterpret_cast<uint4 *>(to + q * job.to.plane + row * job.to.ld + col) = make_uint4(w[q][0], w[q][1], w[q][2], w[q][3]);
    }
}

// ---- shares of a split contraction, added in their order --------------------------------------------------------------------------
struct ShareArgs {
    const float *partial;
    int splits, N;
    long long M;
    void *out0, *out1;
    long long rows0, row1, rows1, ld_out;
    const void *bias;
};
template <class T>
__global__ void __launch_bounds__(256) share_sum_kernel(const ShareArgs p)
{
    grid_launch_dependents();
    grid_dependency_wait();
    const long long all = p.M * p.N;
    for (long long at = (long long)blockIdx.x * 256 + threadIdx.x; at < all; at += (long long)gridDim.x * 256) {
        const long long row = at / p.N;
        const int col = (int)(at - row * p.N);
        T *to;
        if (row < p.rows0) to = static_cast<T *>(p.out0) + row * p.ld_out;
        else if (row >= p.row1 && row < p.row1 + p.rows1) to = static_cast<T *>(p.out1) + (row - p.row1) * p.ld_out;
        else continue;
        float t = 0.f;
#pragma unroll 4
        for (int s = 0; s < p.splits; ++s) t += p.partial[s * all + at];
        if (p.bias != nullptr) t += to_float(static_cast<const T *>(p.bias)[col]);
        to[col] = from_float<T>(t);
    }
}

// ---- sums of columns (the biases' gradients) --------------------------------------------------------------------------------------
// Shares of the rows of a matrix: a block's eight warps take rows in turn, a lane VEC columns, and add up at the end.
template <class T, int VEC>
__global__ void __launch_bounds__(256) column_share_kernel(const T *x, long long rows, int cols, float *partial)
{
    __shared__ float part[8][32 * VEC];
    grid_launch_dependents();
    grid_dependency_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, col = (blockIdx.x * 32 + lane) * VEC;
    const long long lo = rows * blockIdx.y / gridDim.y, hi = rows * (blockIdx.y + 1) / gridDim.y;
    float sum[VEC], low[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) sum[e] = low[e] = 0.f;
    if (col < cols) {
#pragma unroll 4
        for (long long n = lo + warp; n < hi; n += 8) {
            float v[VEC];
            load_values<T, VEC>(x + n * cols + col, v);
#pragma unroll
            for (int e = 0; e < VEC; ++e) add_compensated(v[e], sum[e], low[e]);
        }
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) part[warp][e * 32 + lane] = sum[e] + low[e];
    __syncthreads();
    for (int i = threadIdx.x; i < 32 * VEC; i += 256) {
        const int at = (blockIdx.x * 32 + (i & 31)) * VEC + (i >> 5);
        float t = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) t += part[w][i];
        if (at < cols) partial[(long long)blockIdx.y * cols + at] = t;
    }
}
// Shares added: to fewer of them (`fewer`, gridDim.y of them), or to the columns' places in the gradients.
template <class T>
__global__ void __launch_bounds__(256) column_sum_kernel(const float *partial, long long shares, int cols, float *fewer, T *out0, int cols0, T *out1, int col1,
                                                         int cols1)
{
    __shared__ float part[8][32];
    grid_launch_dependents();
    grid_dependency_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, col = blockIdx.x * 32 + lane;
    const long long lo = shares * blockIdx.y / gridDim.y, hi = shares * (blockIdx.y + 1) / gridDim.y;
    float t = 0.f;
    if (col < cols) {
#pragma unroll 8
        for (long long s = lo + warp; s < hi; s += 8) t += partial[s * cols + col];
    }
    part[warp][lane] = t;
    __syncthreads();
    if (warp > 0 || col >= cols) return;
#pragma unroll
    for (int w = 1; w < 8; ++w) t += part[w][lane];
    if (fewer != nullptr) fewer[(long long)blockIdx.y * cols + col] = t;
    else if (col < cols0) { if (out0 != nullptr) out0[col] = from_float<T>(t); }
    else if (col >= col1 && col < col1 + cols1) { if (out1 != nullptr) out1[col - col1] = from_float<T>(t); }
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
int launch_tiles(const Params &p, bool chained, cudaStream_t s)
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
    const long long tiles = (long long)p.m_tiles * p.n_tiles * p.splits;
    cfg.gridDim = dim3((unsigned)std::min<long long>(PAIR ? 2 * tiles : tiles, blocks));
    cfg.numAttrs = chained && chained_launches_enabled() ? 2 : 1;
    if (cudaLaunchKernelEx(&cfg, tile_kernel<T, MODE, TN, PAIR>, p) != cudaSuccess) return launch_status("tile_kernel");
    return launch_status("tile_kernel");
}

// Blocks of a grid-stride kernel over `work` units of one thread each.
unsigned stride_blocks(long long work) { return (unsigned)std::max(1ll, std::min((work + 255) / 256, (long long)sm_count() * 8)); }

// C (M, N) = sum over parts of A B^T; where splitting pays, float32 shares through `partial`.
struct Linear {
    Operand a[2], b[2];
    bool a_across[2], b_across[2];
    int parts;
    long long K[2];
    long long M;
    int N;
    void *out0, *out1;
    long long rows0, row1, rows1, ld_out;
    const void *bias;
};

int blocks_of(long long K) { return (int)((K + TK - 1) / TK); }

// Width of the tiles, one block or a pair of them to a tile, and number of shares: the cheapest of the kernel's rounds (blocks of the
// contraction, and what a tile costs beside them) and of the shares' way through memory.  Unit: 256 clocks, the products of
// 128 x 128 x 64 values of 16 bits.
struct Cut {
    int tn;
    bool pair;
    int splits;
};
template <class T>
Cut linear_cut(long long M, int N, int blocks)
{
    // a block of the contraction of a 16-bit type: its products, or (tiles of one block) what L2 delivers; of float32: six products
    struct Kind { int tn; bool pair; double one, six; };
    constexpr Kind kinds[] = {{256, true, 2.0, 12.5}, {128, true, 1.15, 6.6}, {128, false, 1.7, 7.2}, {64, false, 1.2, 4.4}};
    constexpr bool wide = pieces_of<T> > 1;
    const double sms = sm_count();
    Cut best{128, false, 1};
    double least = 1e300;
    for (const Kind &k : kinds) {
        const double tiles = (double)((M + (k.pair ? 255 : 127)) / (k.pair ? 256 : 128)) * ((N + k.tn - 1) / k.tn);
        for (int sp = 1; sp <= 64 && sp <= blocks; sp = sp < 4 ? sp + 1 : sp + sp / 4) {
            const double rounds = std::ceil(tiles * sp / (k.pair ? std::floor(sms / 2) : sms));
            // a tile's start and the last one's epilogue: some 8 units; shares: a launch, and 8 bytes a value at 13 KB a unit
            const double cost = rounds * std::ceil((double)blocks / sp) * (wide ? k.six : k.one) + 8.0 + 3.0 * rounds +
                                (sp > 1 ? 16.0 + (double)sp * M * N * 8.0 / 1e6 : 0.0);
            if (cost < least * 0.99) {
                least = cost;
                best = {k.tn, k.pair, sp};
            }
        }
    }
    return best;
}

template <class T>
size_t linear_partial(long long M, int N, int blocks)
{
    const Cut c = linear_cut<T>(M, N, blocks);
    return c.splits > 1 ? (size_t)c.splits * M * N : 0;
}

template <class T>
int run_linear(const Linear &l, float *partial, cudaStream_t s)
{
    Params p{};
    p.blocks0 = blocks_of(l.K[0]);
    p.blocks = p.blocks0 + (l.parts > 1 ? blocks_of(l.K[1]) : 0);
    const Cut cut = linear_cut<T>(l.M, l.N, p.blocks);
    for (int i = 0; i < l.parts; ++i) {
        p.a_across[i] = l.a_across[i];
        p.b_across[i] = l.b_across[i];
        int rc = encode<T>(&p.a[i], l.a[i].x, l.a[i].rows, l.a[i].cols, l.a_across[i] ? TK : TM);
        if (rc == CF_OK) rc = encode<T>(&p.b[i], l.b[i].x, l.b[i].rows, l.b[i].cols, l.b_across[i] ? TK : cut.pair ? cut.tn / 2 : cut.tn);
        if (rc != CF_OK) return rc;
    }
    p.M = l.M;
    p.N = l.N;
    const int tm = cut.pair ? 2 * TM : TM;
    p.m_tiles = (int)((l.M + tm - 1) / tm);
    p.n_tiles = (l.N + cut.tn - 1) / cut.tn;
    p.splits = cut.splits;
    p.out0 = l.out0; p.out1 = l.out1;
    p.rows0 = l.rows0; p.row1 = l.row1; p.rows1 = l.rows1; p.ld_out = l.ld_out;
    p.bias = l.bias;
    p.partial = cut.splits > 1 ? partial : nullptr;
    p.status = wait_status();
    const int rc = cut.tn == 256 ? launch_tiles<T, LINEAR, 256, true>(p, true, s) : cut.pair ? launch_tiles<T, LINEAR, 128, true>(p, true, s) :
                   cut.tn == 128 ? launch_tiles<T, LINEAR, 128, false>(p, true, s) : launch_tiles<T, LINEAR, 64, false>(p, true, s);
    if (rc != CF_OK || cut.splits == 1) return rc;
    const ShareArgs sum{partial, cut.splits, l.N, l.M, l.out0, l.out1, l.rows0, l.row1, l.rows1, l.ld_out, l.bias};
    if (launch_chained(share_sum_kernel<T>, dim3(stride_blocks(l.M * l.N)), dim3(256), 0, s, true, sum) != cudaSuccess) return launch_status("share_sum_kernel");
    return launch_status("share_sum_kernel");
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
        size_t floats = 0;
        if (!backward) {
            floats = linear_partial<T>(d.N, (int)d.D, blocks_of(d.F));
        } else {
            P *g = c.take<P>((size_t)NP * d.N * 2 * Fp);
            dg = {{g, 2 * Fp, d.N * 2 * Fp}, d.N, d.F};
            du = {{g ? g + Fp : g, 2 * Fp, d.N * 2 * Fp}, d.N, d.F};
            const int rows = blocks_of(d.N);
            floats = std::max<size_t>({linear_partial<T>(d.N, (int)d.D, 2 * blocks_of(d.F)), linear_partial<T>(2 * Fp, (int)d.D, rows),
                               linear_partial<T>(d.D, (int)d.F, rows), (size_t)(COLUMN_SHARES * std::max<long long>(2 * Fp, d.D))});
            sums = c.take<float>((size_t)((d.N + 31) / 32) * 2 * Fp);
        }
        partial = c.take<float>(floats);
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
    Params p{};
    // Tiles of pairs (256 x 128; backward in three pieces, whose sums must fit registers, 256 x 64) or of single blocks (128 x 64): the
    // cheaper by rounds times products, single blocks' bound by L2 (16 bits).
    const int pair_tn = wide && backward ? 64 : 128;
    const double sms = sm_count();
    auto rounds = [&](int tm, int tn, double at_once) { return std::ceil((double)((d.N + tm - 1) / tm) * ((d.F + tn - 1) / tn) / at_once); };
    const double blocks = blocks_of(d.D);
    const bool pair = rounds(256, pair_tn, std::floor(sms / 2)) * pair_tn * (blocks + 2) < rounds(128, 64, sms) * 64 * (blocks + 2) * (wide ? 1.1 : 1.4);
    const int tn = pair ? pair_tn : 64, tm = pair ? 2 * TM : TM;
    const int of_x = backward ? 1 : 0;
    p.blocks0 = blocks_of(d.D);
    p.blocks = backward ? 2 * p.blocks0 : p.blocks0;
    int rc = encode<T>(&p.a[of_x], plan.x.x, d.N, d.D, TM);
    if (rc == CF_OK) rc = encode<T>(&p.b[1], plan.wg.x, d.F, d.D, tn);
    if (rc == CF_OK) rc = encode<T>(&p.b[2], plan.wu.x, d.F, d.D, tn);
    if (backward) {
        if (rc == CF_OK) rc = encode<T>(&p.a[0], plan.gy.x, d.N, d.D, TM);
        if (rc == CF_OK) rc = wide ? encode<T>(&p.b[0], plan.wd.x, d.F, d.D, pair ? tn / 2 : tn) : encode<T>(&p.b[0], plan.wd.x, d.D, d.F, TK);
        p.b_across[0] = !wide;
        p.dg = plan.dg.x;
        p.du = plan.du.x;
        p.sums = sums ? plan.sums : nullptr;
    }
    if (rc != CF_OK) return rc;
    p.m_tiles = (int)((d.N + tm - 1) / tm);
    p.n_tiles = (int)((d.F + tn - 1) / tn);
    p.splits = 1;
    p.M = d.N;
    p.N = (int)d.F;
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
    return run_linear<T>(l, plan.partial, s);
}

// The shares of columns in `from` (through `fewer` where they are many) to their places.
template <class T>
int column_sums(const float *from, long long shares, int cols, float *fewer, T *out0, int cols0, T *out1, int col1, int cols1, cudaStream_t s)
{
    const unsigned groups = (unsigned)(cols + 31) / 32;
    if (shares > 256) {
        const unsigned to = (unsigned)std::min<long long>(COLUMN_SHARES, shares / 64);
        launch_chained(column_sum_kernel<T>, dim3(groups, to), dim3(256), 0, s, true, from, shares, cols, fewer, out0, cols0, out1, col1, cols1);
        from = fewer;
        shares = to;
    }
    launch_chained(column_sum_kernel<T>, dim3(groups), dim3(256), 0, s, true, from, shares, cols, static_cast<float *>(nullptr), out0, cols0, out1, col1, cols1);
    return launch_status("column_sum_kernel");
}

template <class T>
int row_sums(const T *x, long long rows, int cols, float *partial, T *out, cudaStream_t s)
{
    constexpr int VEC = 16 / sizeof(T);
    const bool wide = cols % VEC == 0 && aligned_to(x, 16);
    const unsigned groups = (unsigned)(cols + (wide ? 32 * VEC : 32) - 1) / (wide ? 32 * VEC : 32);
    const unsigned shares = (unsigned)std::max(1ll, std::min<long long>(COLUMN_SHARES, rows / 32));
    if (wide) launch_chained(column_share_kernel<T, VEC>, dim3(groups, shares), dim3(256), 0, s, true, x, rows, cols, partial);
    else launch_chained(column_share_kernel<T, 1>, dim3(groups, shares), dim3(256), 0, s, true, x, rows, cols, partial);
    return column_sums<T>(partial, shares, cols, nullptr, out, cols, nullptr, cols, 0, s);
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
    if (g.x) {
        Linear l{};
        l.a[0] = plan.dg; l.b[0] = plan.wg;
        l.a[1] = plan.du; l.b[1] = plan.wu;
        l.b_across[0] = l.b_across[1] = true;
        l.parts = 2;
        l.K[0] = l.K[1] = F;
        l.M = d.N; l.N = D;
        l.out0 = g.x; l.rows0 = d.N; l.row1 = d.N; l.ld_out = D;
        if ((rc = run_linear<T>(l, plan.partial, s)) != CF_OK) return rc;
    }
    if (g.w_gate || g.w_up) {  // one product for both: rows [0, F) and [Fp, Fp + F)
        Linear l{};
        l.a[0] = {plan.dg.x, d.N, 2 * Fp}; l.b[0] = plan.x;
        l.a_across[0] = l.b_across[0] = true;
        l.parts = 1;
        l.K[0] = d.N;
        l.M = 2 * Fp; l.N = D;
        l.out0 = g.w_gate; l.rows0 = g.w_gate ? F : 0;
        l.out1 = g.w_up; l.row1 = Fp; l.rows1 = g.w_up ? F : 0;
        l.ld_out = D;
        if ((rc = run_linear<T>(l, plan.partial, s)) != CF_OK) return rc;
    }
    if (g.w_down) {
        Linear l{};
        l.a[0] = plan.gy; l.b[0] = plan.h;
        l.a_across[0] = l.b_across[0] = true;
        l.parts = 1;
        l.K[0] = d.N;
        l.M = D; l.N = F;
        l.out0 = g.w_down; l.rows0 = D; l.row1 = D; l.ld_out = F;
        if ((rc = run_linear<T>(l, plan.partial, s)) != CF_OK) return rc;
    }
    if (g.b_gate || g.b_up) {
        rc = column_sums<T>(plan.sums, (d.N + 31) / 32, (int)(2 * Fp), plan.partial, static_cast<T *>(g.b_gate), F, static_cast<T *>(g.b_up), (int)Fp, F, s);
        if (rc != CF_OK) return rc;
    }
    if (g.b_down) rc = row_sums<T>(static_cast<const T *>(g.gy), d.N, D, plan.partial, static_cast<T *>(g.b_down), s);
    return rc;
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
