// The tile products of the gated feed-forward on the fifth-generation tensor cores, in three modes:
//
//   LINEAR        C = A0 B0^T [+ A1 B1^T]                       epilogue: bias, stored in the type of the call; of a split contraction
//                                                               float32 shares, added by whoever brings a tile's last.  Up to three
//                                                               products in one launch
//   GLU_FORWARD   g = X Wg^T, u = X Wu^T                        epilogue: h = act(g + bg) (u + bu)
//   GLU_BACKWARD  dh = Gy Wd, then the same                     epilogue: h, dg = dh u act'(g), du = dh act(g), sums of columns of 32 rows
//
// A block holds a 128-row tile of each accumulator in tensor memory, TN columns wide, and walks the contraction in blocks of 64: one
// thread keeps STAGES of them in flight by TMA (128-byte swizzle; either order of an operand, its contraction running along or across
// its rows), one thread issues tcgen05.mma, sixteen warps take the accumulators.  PAIR: two blocks of a cluster share their products
// (cta_group::2, 256 rows): each fetches half of B, which halves what a block of the contraction moves from L2 (32 KB per 128 x 256
// products of 64; the tiles of one block are bound by that).  The grid is as large as the GPU and every block walks tiles, so that a
// tile's epilogue runs beside the next one's products: two sets of accumulators; GLU_BACKWARD of 16-bit types, whose set is 384 of
// the 512 columns, has two of dh alone and computes the next tile's dh beside the epilogue.
//
// 16-bit types: one product per pair of blocks; rows of 64 values are 128 bytes; a contraction stays in its accumulator, in shares short
// enough for what that loses (find_cut).  float32: an operand is the sum of three bfloat16
// pieces (24 bits of values from 2^-109 on, of smaller ones what lies above 2^-133), made once by a packing kernel or by the epilogue
// that produces it, and a product is six: piece 0 with 0, 1, 2, piece 1 with 0, 1 and piece 2 with 0 (what is left out is 2^-26 of a
// product).  What overflows is an infinity, or no number where it meets a value beyond 256, whose second piece may have the other sign.
// The tensor core's running sums lose low bits with every instruction, so that with three pieces each block of 64 has accumulators of
// its own, smallest products first, and the sums over blocks are added in registers: errors are those of float32 sums (3e-7 relative at
// 512 terms).  The projections of models of up to 128 features, two blocks, stay in their accumulators, the small products of both
// before the large ones: the epilogue then takes a tile at once, beside the next one's products (backward of 133,120 rows, 128 x 512:
// 602 -> 455 us).
//
// All waits are bounded (tc5::mbar_wait); one that runs out ends the block after its copies and products in flight.
#pragma once
#include <cuda.h>

#include <type_traits>

#include "common.cuh"
#include "tc5.cuh"
#include "values.cuh"

namespace cf {
namespace tile {

enum Mode { LINEAR = 0, GLU_FORWARD = 1, GLU_BACKWARD = 2 };
enum Activation { SILU = 0, GELU = 1, RELU = 2 };

constexpr int TM = 128, TK = 64;
constexpr int EPILOGUE_WARPS = 16, THREADS = (EPILOGUE_WARPS + 2) * 32;

template <class T> constexpr int pieces_of = sizeof(T) == 4 ? 3 : 1;
template <class T> struct Piece { using type = T; };
template <> struct Piece<float> { using type = __nv_bfloat16; };

// Rows of pieces: value (row, col) of piece i at base + i * plane + row * ld + col.
struct Planes {
    void *base;
    long long ld, plane;
};

// One product.  LINEAR: a[0] with b[0], a[1] with b[1]; GLU: x with b[1] (gate) and b[2] (up), backward: gy = a[0] with b[0] (down),
// x = a[1].
struct Problem {
    CUtensorMap a[2], b[3];
    int a_across[2], b_across[2];  // per part: the contraction runs across the rows of the operand
    int blocks0, blocks;      // of the contraction: of the first part, of both
    int m_tiles, n_tiles, splits;  // m_tiles: of 128 rows, or 256 of a pair
    int N;
    long long M, tiles;       // tiles = m_tiles n_tiles splits
    // LINEAR: rows [0, rows0) to out0, rows [row1, row1 + rows1) to out1
    void *out0, *out1;
    long long rows0, row1, rows1, ld_out;
    int transposed;           // out0 (N, rows0): its rows are the columns
    const void *bias;
    // splits > 1: every share of a tile, and how many of a warp's part of it are there (zero before); who brings the last adds them
    float *partial;
    unsigned *tickets;
};

template <int COUNT>
struct Params {
    Problem q[COUNT];
    int count;
    unsigned *clear;          // words that GLU sets to zero, for the kernels behind it
    int clear_words;
    unsigned *status;
    // GLU
    const void *bias_gate, *bias_up;
    int act;
    int padded;               // columns that h, dg and du have memory for, a multiple of 16
    Planes h, dg, du;
    float *sums;              // or null: (32 rows each, 2 padded) sums of the columns of dg and du
};
constexpr int LINEAR_COUNT = 3;  // products that one launch may have
constexpr int WHOLE = 2;  // blocks of a contraction that float32 accumulators keep whole (more of them were not measured)
template <int MODE> using ParamsOf = Params<MODE == LINEAR ? LINEAR_COUNT : 1>;

template <class T, int MODE, int TN, bool PAIR>
struct Shape {
    static constexpr int NP = pieces_of<T>;
    // rows of B that a block fetches per block of the contraction: of both projections, of a single matrix
    static constexpr int ROWS_GU = PAIR ? TN : 2 * TN, ROWS_ONE = PAIR ? TN / 2 : TN, ROWS = MODE == LINEAR ? ROWS_ONE : ROWS_GU;
    static constexpr int ACCS = MODE == LINEAR ? 1 : MODE == GLU_FORWARD ? 2 : 3;
    static constexpr int A_PIECE = TM * TK * 2, B_PIECE = ROWS * TK * 2;
    static constexpr int STAGE = NP * (A_PIECE + B_PIECE);
    static constexpr int ROOM = 220 * 1024;
    static constexpr int STAGES = ROOM / STAGE < 8 ? ROOM / STAGE : 8;
    static constexpr int WIDTH = ACCS * TN;                               // columns of a set of accumulators: g, u, dh
    static constexpr bool SHARED_SET = NP == 1 && MODE == GLU_BACKWARD;   // one set, two of dh behind it
    static constexpr int SETS = SHARED_SET ? 1 : 2;
    static constexpr int USED = SHARED_SET ? 4 * TN : 2 * WIDTH;
    static constexpr int TMEM = USED <= 64 ? 64 : USED <= 128 ? 128 : USED <= 256 ? 256 : 512;
    static constexpr int MISC = STAGES * STAGE, BIAS = MISC + 256;
    static constexpr int SMEM = BIAS + EPILOGUE_WARPS * 128;
    static_assert(STAGES >= 2 && USED <= 512, "tile");
};

// ---- activations: value and derivative ---------------------------------------------------------------------------------------
struct Gate {
    float a, da;
};
template <int ACT>
__device__ __forceinline__ Gate gate_of(float g)
{
    if constexpr (ACT == SILU) {
        const float p = __fdividef(1.f, 1.f + expf(-g));
        return {g * p, p * (1.f + g * (1.f - p))};
    } else if constexpr (ACT == GELU) {
        const float p = 0.5f * (1.f + erff(g * 0.70710678118654752f));
        return {g * p, p + g * expf(-0.5f * g * g) * 0.39894228040143268f};
    } else {
        // (a value that is no number stays one)
        return {g > 0.f || g != g ? g : 0.f, g > 0.f ? 1.f : 0.f};
    }
}

// Two values in one word, the first in the lower half; what would round to an infinity, infinities too, is the largest finite value.
__device__ __forceinline__ uint32_t pack_two_finite(float a, float b)
{
    uint32_t w;
    asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(b), "f"(a));
    return w;
}

// The three bfloat16 pieces of 2 COUNT values, as words of two.  The first two are finite: the largest floats keep all their bits, and
// an infinity is in the third piece, which meets first pieces only - a first piece would meet zeros and pieces of either sign.
template <int COUNT>
__device__ __forceinline__ void split_words(const float (&v)[2 * COUNT], uint32_t (&w)[3][COUNT])
{
#pragma unroll
    for (int i = 0; i < COUNT; ++i) {
        float a = v[2 * i], b = v[2 * i + 1];
#pragma unroll
        for (int p = 0; p < 3; ++p) {
            w[p][i] = p < 2 ? pack_two_finite(a, b) : pack_two<__nv_bfloat16>(a, b);
            const float2 f = unpack_two<__nv_bfloat16>(w[p][i]);
            a -= f.x;
            b -= f.y;
        }
    }
}

// 16 neighbours of a row into its planes (32 bytes of each: a sector).
template <class T>
__device__ __forceinline__ void store_planes(const Planes &to, long long row, int col, const float (&v)[16])
{
    constexpr int NP = pieces_of<T>;
    using P = typename Piece<T>::type;
    P *at = static_cast<P *>(to.base) + row * to.ld + col;
    uint32_t w[NP][8];
    if constexpr (NP == 3) {
        split_words(v, w);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[0][i] = pack_two<P>(v[2 * i], v[2 * i + 1]);
    }
#pragma unroll
    for (int p = 0; p < NP; ++p) store_32(at + p * to.plane, w[p]);
}

// 16 neighbours of a row, on 32 bytes.
template <class T>
__device__ __forceinline__ void store_run(T *to, const float (&v)[16])
{
    uint32_t w[8];
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(v[8 * half + i]);
            store_32(to + 8 * half, w);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = pack_two<T>(v[2 * i], v[2 * i + 1]);
        store_32(to, w);
    }
}

// 16 rows by 16 columns, a row per lane of half a warp, to a column per lane.
__device__ __forceinline__ void transpose_16(float (&v)[16], int lane)
{
#pragma unroll
    for (int s = 8; s > 0; s >>= 1)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if (i & s) continue;
            const bool upper = lane & s;
            const float got = __shfl_xor_sync(FULL, upper ? v[i] : v[i + s], s);
            if (upper) v[i] = got;
            else v[i + s] = got;
        }
}

// A lane's bias of 16 columns: of the first (lanes 0 to 15) and the second vector.
template <class T>
__device__ __forceinline__ float lane_bias(const void *first, const void *second, int col, int N, int lane)
{
    const T *b = static_cast<const T *>(lane < 16 ? first : second);
    const int at = col + (lane & 15);
    return b != nullptr && at < N ? to_float(b[at]) : 0.f;
}
__device__ __forceinline__ void add_16(const float *b, float (&v)[16])
{
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float4 w = reinterpret_cast<const float4 *>(b)[i];
        v[4 * i] += w.x; v[4 * i + 1] += w.y; v[4 * i + 2] += w.z; v[4 * i + 3] += w.w;
    }
}

// Sums of 16 columns over a warp's 32 rows by halving: lanes 2 c and 2 c + 1 end with column c.
__device__ __forceinline__ float column_sum(const float (&v)[16], int lane)
{
    float a[8], b[4], c[2];
    const bool b4 = lane & 16, b3 = lane & 8, b2 = lane & 4, b1 = lane & 2;
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = (b4 ? v[8 + i] : v[i]) + __shfl_xor_sync(FULL, b4 ? v[i] : v[8 + i], 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = (b3 ? a[4 + i] : a[i]) + __shfl_xor_sync(FULL, b3 ? a[i] : a[4 + i], 8);
#pragma unroll
    for (int i = 0; i < 2; ++i) c[i] = (b2 ? b[2 + i] : b[i]) + __shfl_xor_sync(FULL, b2 ? b[i] : b[2 + i], 4);
    const float d = (b1 ? c[1] : c[0]) + __shfl_xor_sync(FULL, b1 ? c[0] : c[1], 2);
    return d + __shfl_xor_sync(FULL, d, 1);
}

// The epilogue of 16 columns of a warp's 32 rows: v[acc][.] are the accumulators' values of this lane's row.
template <class T, int MODE, int ACT>
__device__ __forceinline__ void finish_glu(const Params<1> &p, long long row, int col, const float *bias, float (&v)[MODE == GLU_FORWARD ? 2 : 3][16])
{
    if (bias != nullptr) {
        add_16(bias, v[0]);
        add_16(bias + 16, v[1]);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const Gate a = gate_of<ACT>(v[0][i]);
        const float u = v[1][i];
        if constexpr (MODE == GLU_BACKWARD) {
            const float dh = v[2][i];
            v[1][i] = dh * a.a;
            v[2][i] = dh * u * a.da;
        }
        v[0][i] = a.a * u;
    }
    if constexpr (MODE == GLU_BACKWARD) {
        if (p.sums != nullptr) {
            const int lane = threadIdx.x & 31;
            const float du = column_sum(v[1], lane), dg = column_sum(v[2], lane);  // (rows behind the last have dh = 0)
            float *to = p.sums + (row >> 5) * (2ll * p.padded) + col + (lane >> 1);
            if ((lane & 1) == 0 && (row & ~31ll) < p.q[0].M) {
                to[0] = dg;
                to[p.padded] = du;
            }
        }
    }
    if (row >= p.q[0].M) return;
    store_planes<T>(p.h, row, col, v[0]);
    if constexpr (MODE == GLU_BACKWARD) {
        store_planes<T>(p.du, row, col, v[1]);
        store_planes<T>(p.dg, row, col, v[2]);
    }
}

// Where a row of the product goes (null: nowhere).
template <class T>
__device__ __forceinline__ T *place_of_row(const Problem &q, long long row)
{
    if (row < q.rows0) return static_cast<T *>(q.out0) + row * q.ld_out;
    if (row >= q.row1 && row < q.row1 + q.rows1) return static_cast<T *>(q.out1) + (row - q.row1) * q.ld_out;
    return nullptr;
}

// 16 columns of a warp's 32 rows; row: this lane's.
template <class T>
__device__ __forceinline__ void finish_linear(const Problem &q, long long row, int col, const float *bias, float (&v)[16])
{
    if (col >= q.N) return;
    const int lane = threadIdx.x & 31;
    if (bias != nullptr) add_16(bias, v);
    if (q.transposed) {  // (a warp's 32 rows are neighbours there)
        if (row >= q.M) return;
        T *to = static_cast<T *>(q.out0) + (long long)col * q.ld_out + row;
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (col + i < q.N) to[i * q.ld_out] = from_float<T>(v[i]);
        return;
    }
    const uintptr_t at = reinterpret_cast<uintptr_t>(q.out0) | reinterpret_cast<uintptr_t>(q.out1) | (uintptr_t)(q.ld_out * sizeof(T));
    if ((at & 31) == 0 && q.N - col >= 16) {
        T *to = row < q.M ? place_of_row<T>(q, row) : nullptr;
        if (to != nullptr) store_run<T>(to + col, v);
        return;
    }
    // rows off 32 bytes, the last columns: value by value, neighbours from neighbouring lanes (a row from each lane touches 32 lines with
    // every store: 26 us instead of 14 for y of 4,999 rows, 201 x 517, float16)
    transpose_16(v, lane);
    const long long first = row - lane + (lane & 16);
    const int c = col + (lane & 15);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        T *to = first + i < q.M ? place_of_row<T>(q, first + i) : nullptr;
        if (to != nullptr && c < q.N) to[c] = from_float<T>(v[i]);
    }
}

template <class T, int MODE, int COUNT>
__device__ __forceinline__ void finish(const ParamsOf<MODE> &p, const Problem &q, long long row, int col, const float *bias, float (&v)[COUNT][16])
{
    if constexpr (MODE == LINEAR) {
        finish_linear<T>(q, row, col, bias, v[0]);
    } else {
        if (col >= q.N) return;
        if (p.act == SILU) finish_glu<T, MODE, SILU>(p, row, col, bias, v);
        else if (p.act == GELU) finish_glu<T, MODE, GELU>(p, row, col, bias, v);
        else finish_glu<T, MODE, RELU>(p, row, col, bias, v);
    }
}

struct Tile {
    int q;  // which product
    int m, n, split;
    int k_lo, k_hi;
};
template <int COUNT>
__device__ __forceinline__ Tile tile_of(const Params<COUNT> &p, long long t)
{
    // (columns run fastest: neighbours share rows of A, which are many, and the whole of B, which is small, stays in L2)
    Tile x;
    x.q = 0;
    if constexpr (COUNT > 1) {
        while (x.q + 1 < p.count && t >= p.q[x.q].tiles) t -= p.q[x.q++].tiles;
    }
    const Problem &q = p.q[x.q];
    const unsigned at = (unsigned)t, n_tiles = q.n_tiles, m_tiles = q.m_tiles;  // (a launch has fewer than 2^31 tiles)
    x.n = (int)(at % n_tiles);
    x.m = (int)(at / n_tiles % m_tiles);
    x.split = (int)(at / n_tiles / m_tiles);
    x.k_lo = (int)((long long)q.blocks * x.split / q.splits);
    x.k_hi = (int)((long long)q.blocks * (x.split + 1) / q.splits);
    return x;
}

template <class T, int MODE, int TN, bool PAIR>
__global__ void __launch_bounds__(THREADS, 1) tile_kernel(const __grid_constant__ ParamsOf<MODE> p)
{
    using namespace tc5;
    using S = Shape<T, MODE, TN, PAIR>;
    constexpr int NP = S::NP, STAGES = S::STAGES, SETS = S::SETS;
    extern __shared__ __align__(1024) unsigned char smem[];
    const uint32_t base = smem_u32(smem), misc = base + S::MISC;
    volatile unsigned *gave_up = reinterpret_cast<volatile unsigned *>(smem + S::MISC + 240);
    auto full = [&](int s) { return misc + 8u * (uint32_t)s; };        // of a pair: the first block's
    auto empty = [&](int s) { return misc + 64u + 8u * (uint32_t)s; };  // either block's
    auto ready = [&](int b) { return misc + 128u + 8u * (uint32_t)b; };  // either block's
    auto taken = [&](int b) { return misc + 144u + 8u * (uint32_t)b; };  // the first block's
    const uint32_t drained = misc + 160u;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = PAIR ? cluster_rank() : 0u;
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) { mbar_init(full(s), 1); mbar_init(empty(s), 1); }
        for (int b = 0; b < SETS; ++b) { mbar_init(ready(b), 1); mbar_init(taken(b), PAIR ? 2 * EPILOGUE_WARPS : EPILOGUE_WARPS); }
        mbar_init(drained, 1);
        *gave_up = 0u;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_smem();
    }
    if (warp == EPILOGUE_WARPS) {
        if constexpr (PAIR) tmem_alloc_pair<S::TMEM>(misc + 232);
        else tmem_alloc<S::TMEM>(misc + 232);
    }
    fence_before();
    __syncthreads();
    if constexpr (PAIR) cluster_sync();
    fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(smem + S::MISC + 232);
    grid_launch_dependents();
    grid_dependency_wait();
    long long tiles = 0;
    for (int i = 0; i < p.count; ++i) tiles += p.q[i].tiles;
    if constexpr (MODE != LINEAR) {
        for (int i = blockIdx.x * THREADS + threadIdx.x; i < p.clear_words; i += gridDim.x * THREADS) p.clear[i] = 0u;
    }
    const long long first_tile = PAIR ? blockIdx.x >> 1 : blockIdx.x, stride = PAIR ? gridDim.x >> 1 : gridDim.x;
    // whether a block of the contraction multiplies with both projections
    // three pieces: whether an accumulator keeps the whole contraction (WHOLE blocks at most), or each block of it goes to registers
    const bool whole = NP > 1 && MODE != LINEAR && p.q[0].blocks0 <= WHOLE;
    auto is_gu = [&](int kb) { return MODE == GLU_FORWARD || (MODE == GLU_BACKWARD && kb >= p.q[0].blocks0); };

    if (warp == EPILOGUE_WARPS + 1) {
        // ---- copies ----
        if (lane == 0) {
            int s = 0;
            uint32_t phase = 1;
            bool ok = true;
            long long sent = 0;
            auto box = [&](uint32_t to, const CUtensorMap *map, int x, int y, int z, uint32_t bar) {
                if constexpr (PAIR) tma_load_3d_pair(to, map, x, y, z, bar);
                else tma_load_3d(to, map, x, y, z, bar);
            };
            auto operand = [&](const CUtensorMap *map, bool across, uint32_t to, int rows, int row, int k, int piece, uint32_t bar) {
                if (!across) {
                    box(to, map, k, row, piece, bar);
                } else {
                    for (int i = 0; i < rows; i += 64) box(to + i * 128u, map, row + i, k, piece, bar);
                }
            };
            for (long long t = first_tile; t < tiles && ok; t += stride) {
                const Tile x = tile_of(p, t);
                const Problem &q = p.q[x.q];
                const int m0 = (PAIR ? 2 * x.m + (int)rank : x.m) * TM, n0 = x.n * TN;
                for (int kb = x.k_lo; kb < x.k_hi; ++kb) {
                    ok = mbar_wait(empty(s), phase, gave_up);
                    if (!ok) break;
                    const int part = kb >= q.blocks0, k = (part ? kb - q.blocks0 : kb) * TK;
                    const bool gu = is_gu(kb);
                    const uint32_t at = base + s * S::STAGE, bt = at + NP * S::A_PIECE;
                    const uint32_t bar = PAIR ? mapa(full(s), 0) : full(s);
                    if (rank == 0)
                        mbar_expect(full(s), (uint32_t)((PAIR ? 2 : 1) * NP * (S::A_PIECE + (gu ? S::ROWS_GU : S::ROWS_ONE) * TK * 2)));
#pragma unroll
                    for (int i = 0; i < NP; ++i) {
                        operand(&q.a[part], q.a_across[part], at + i * S::A_PIECE, TM, m0, k, i, bar);
                        const uint32_t bi = bt + i * S::B_PIECE;
                        if (gu) {
                            if (PAIR) {
                                operand(&q.b[1 + rank], false, bi, TN, n0, k, i, bar);
                            } else {
                                operand(&q.b[1], false, bi, TN, n0, k, i, bar);
                                operand(&q.b[2], false, bi + TN * TK * 2, TN, n0, k, i, bar);
                            }
                        } else {
                            operand(&q.b[part], q.b_across[part], bi, S::ROWS_ONE, n0 + (int)rank * S::ROWS_ONE, k, i, bar);
                        }
                    }
                    ++sent;
                    if (++s == STAGES) { s = 0; phase ^= 1u; }
                }
            }
            // every stage given back: a commit arrives in both blocks of a pair, and in neither behind its end
            for (int e = 0; e < STAGES && ok; ++e) ok = mbar_wait(empty(e), e < s ? phase ^ 1u : phase, gave_up);
            if (!ok && rank == 0) {  // the copies in flight land before the block goes (and its pair: the cluster leaves together)
                unsigned mine = 0u;
                for (int i = 0; i < STAGES && i < sent; ++i) {
                    if (--s < 0) { s = STAGES - 1; phase ^= 1u; }
                    mbar_wait(full(s), phase ^ 1u, &mine);
                }
            }
        }
    } else if (warp == EPILOGUE_WARPS) {
        // ---- products ----
        if (lane == 0 && rank == 0) {
            constexpr int AB = std::is_same<typename Piece<T>::type, __half>::value ? 0 : 1, IM = PAIR ? 2 * TM : TM;
            auto mma = [&](uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
                if constexpr (PAIR) mma_f16_pair(d, a, b, idesc, accumulate);
                else mma_f16(d, a, b, idesc, accumulate);
            };
            auto commit = [&](uint32_t bar) {
                if constexpr (PAIR) mma_commit_pair(bar);
                else mma_commit(bar);
            };
            int s = 0, b = 0, dh_set = 0;
            uint32_t phase = 0, set_phase = 1;
            bool ok = true;
            for (long long t = first_tile; t < tiles && ok; t += stride) {
                const Tile x = tile_of(p, t);
                const Problem &q = p.q[x.q];
                for (int kb = x.k_lo; kb < x.k_hi; ++kb) {
                    const int part = kb >= q.blocks0;
                    const bool gu = is_gu(kb);
                    const bool starts = kb == x.k_lo || (MODE == GLU_BACKWARD && kb == q.blocks0);  // a part
                    const bool clear = NP == 1 ? starts : !whole || starts;  // the first block of an accumulator
                    // (where the sets of dh lie behind a shared one, that of the tile before last has been taken: see the wait below)
                    if (S::SHARED_SET ? clear && gu : NP > 1 && !whole ? true : kb == x.k_lo) {
                        ok = mbar_wait(taken(b), set_phase, gave_up);
                        if (!ok) break;
                        fence_after();
                    }
                    ok = mbar_wait(full(s), phase, gave_up);
                    if (!ok) break;
                    fence_after();
                    const uint32_t d = tmem + (S::SHARED_SET ? (gu ? 0u : (2u + dh_set) * TN) : (uint32_t)(b * S::WIDTH + (MODE == GLU_BACKWARD && !gu ? 2 * TN : 0)));
                    const bool aa = q.a_across[part], ba = !gu && q.b_across[part];
                    const uint32_t idesc = (gu ? instr_desc<IM, MODE == LINEAR ? TN : 2 * TN, AB, false>() : instr_desc<IM, TN, AB, false>()) |
                                           (aa ? 1u << 15 : 0u) | (ba ? 1u << 16 : 0u);
                    // a step of 16 along the contraction: 32 bytes of a row, or 16 rows; panels of 64 across it lie 8 KB apart
                    const uint32_t a_step = (aa ? 2048 : 32) >> 4, b_step = (ba ? 2048 : 32) >> 4;
                    const uint32_t at = base + s * S::STAGE, bt = at + NP * S::A_PIECE;
                    const uint64_t a0 = smem_desc(at, 8192, 1024), b0 = smem_desc(bt, 8192, 1024);
                    constexpr uint32_t AP = S::A_PIECE >> 4, BP = S::B_PIECE >> 4;
                    if constexpr (NP == 1) {
#pragma unroll
                        for (int ks = 0; ks < TK / 16; ++ks) mma(d, a0 + ks * a_step, b0 + ks * b_step, idesc, !(clear && ks == 0));
                    } else {
                        // small products first; of a whole contraction those of both blocks, before the large ones of either
                        auto small = [&](uint64_t ak0, uint64_t bk0, bool first) {
#pragma unroll
                            for (int ks = 0; ks < TK / 16; ++ks) {
                                const uint64_t ak = ak0 + ks * a_step, bk = bk0 + ks * b_step;
                                mma(d, ak + 2 * AP, bk, idesc, !(first && ks == 0));
                                mma(d, ak, bk + 2 * BP, idesc, true);
                                mma(d, ak + AP, bk + BP, idesc, true);
                            }
#pragma unroll
                            for (int ks = 0; ks < TK / 16; ++ks) {
                                const uint64_t ak = ak0 + ks * a_step, bk = bk0 + ks * b_step;
                                mma(d, ak + AP, bk, idesc, true);
                                mma(d, ak, bk + BP, idesc, true);
                            }
                        };
                        auto large = [&](uint64_t ak0, uint64_t bk0) {
#pragma unroll
                            for (int ks = 0; ks < TK / 16; ++ks) mma(d, ak0 + ks * a_step, bk0 + ks * b_step, idesc, true);
                        };
                        small(a0, b0, clear);
                        if (whole && starts && q.blocks0 == 2) {
                            int s2 = s + 1;
                            uint32_t phase2 = phase;
                            if (s2 == STAGES) { s2 = 0; phase2 ^= 1u; }
                            ok = mbar_wait(full(s2), phase2, gave_up);
                            if (!ok) break;
                            fence_after();
                            const uint64_t a1 = smem_desc(base + s2 * S::STAGE, 8192, 1024), b1 = smem_desc(base + s2 * S::STAGE + NP * S::A_PIECE, 8192, 1024);
                            small(a1, b1, false);
                            large(a0, b0);
                            commit(empty(s));
                            large(a1, b1);
                            s = s2;
                            phase = phase2;
                            ++kb;
                        } else {
                            large(a0, b0);
                        }
                    }
                    commit(empty(s));
                    if (++s == STAGES) { s = 0; phase ^= 1u; }
                    if ((NP > 1 && !whole) || kb == x.k_hi - 1) {
                        commit(ready(b));
                        if (++b == SETS) { b = 0; set_phase ^= 1u; }
                    }
                }
                dh_set ^= 1;
            }
            if (!ok) {  // the instructions issued so far
                unsigned mine = 0u;
                if constexpr (PAIR) mma_commit_pair(drained, 1);  // (here only: the other block has no wait for it)
                else mma_commit(drained);
                mbar_wait(drained, 0, &mine);
            }
        }
    } else {
        // ---- epilogue: warp w has rows 32 (w % 4) .. + 31 of the tile and a quarter of its columns ----
        constexpr int SHARE = TN / (EPILOGUE_WARPS / 4), CHUNKS = SHARE / 16;
        const int first = (warp >> 2) * SHARE;
        const uint32_t lanes = tmem + ((uint32_t)(warp & 3) << 21) + first;
        float *bias_16 = reinterpret_cast<float *>(smem + S::BIAS) + warp * 32;
        auto give_back = [&](int b) {
            fence_before();
            __syncwarp();
            if (lane == 0) {
                if constexpr (PAIR) mbar_arrive_at(mapa(taken(b), 0));
                else mbar_arrive(taken(b));
            }
        };
        int b = 0, dh_set = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (long long t = first_tile; t < tiles && ok; t += stride) {
            const Tile x = tile_of(p, t);
            const Problem &q = p.q[x.q];
            const void *bias_a = MODE == LINEAR ? q.bias : p.bias_gate, *bias_b = MODE == LINEAR ? nullptr : p.bias_up;
            const bool biased = bias_a != nullptr || bias_b != nullptr;
            const bool split = MODE == LINEAR && q.splits > 1;
            // a warp's part of a tile's shares: 16 columns of a lane's row as four vectors, lanes as neighbours
            const long long mine = ((long long)x.m * q.n_tiles + x.n) * (PAIR ? 2 : 1) + rank;
            float4 *shares = reinterpret_cast<float4 *>(q.partial) + ((mine * q.splits * EPILOGUE_WARPS + warp) * CHUNKS * 4) * 32 + lane;
            const long long per_share = (long long)EPILOGUE_WARPS * CHUNKS * 4 * 32;
            auto put_share = [&](int c, const float (&v)[16]) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    __stcg(shares + x.split * per_share + (c * 4 + i) * 32, make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]));
            };
            const long long row = ((long long)(PAIR ? 2 * x.m + rank : x.m)) * TM + (warp & 3) * 32 + lane;
            const int col = x.n * TN + first;
            float bias[CHUNKS];
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c) bias[c] = biased ? lane_bias<T>(bias_a, bias_b, col + c * 16, q.N, lane) : 0.f;
            auto place_bias = [&](int c) -> const float * {
                if (!biased) return nullptr;
                __syncwarp();
                bias_16[lane] = bias[c];
                __syncwarp();
                return bias_16;
            };
            if (NP == 1 || whole) {
                ok = mbar_wait(ready(b), phase, gave_up);
                ok = __all_sync(FULL, ok);
                if (!ok) break;
                fence_after();
#pragma unroll
                for (int c = 0; c < CHUNKS; ++c) {
                    float v[S::ACCS][16];
                    const uint32_t at = lanes + b * S::WIDTH + c * 16;
                    // (dh is the third accumulator: two or three widths behind the first)
                    tmem_load_rows16<S::ACCS>(at, TN, v, S::SHARED_SET ? dh_set * TN : 0);
                    if (c == CHUNKS - 1) give_back(b);
                    if (split) put_share(c, v[0]);
                    else finish<T, MODE>(p, q, row, col + c * 16, place_bias(c), v);
                }
                if (++b == SETS) { b = 0; phase ^= 1u; }
                dh_set ^= 1;
            } else if constexpr (NP > 1) {
                float sum[CHUNKS][S::ACCS][16];
#pragma unroll
                for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
                    for (int a = 0; a < S::ACCS; ++a)
#pragma unroll
                        for (int i = 0; i < 16; ++i) sum[c][a][i] = 0.f;
                for (int kb = x.k_lo; kb < x.k_hi; ++kb) {
                    ok = mbar_wait(ready(b), phase, gave_up);
                    ok = __all_sync(FULL, ok);
                    if (!ok) break;
                    fence_after();
                    const uint32_t at = lanes + b * S::WIDTH;
                    if (MODE == GLU_BACKWARD && kb < q.blocks0) {
#pragma unroll
                        for (int c = 0; c < CHUNKS; ++c) {
                            float v[1][16];
                            tmem_load_rows16<1>(at + 2 * TN + c * 16, TN, v, 0);
#pragma unroll
                            for (int i = 0; i < 16; ++i) sum[c][S::ACCS - 1][i] += v[0][i];
                        }
                    } else {
                        constexpr int NOW = MODE == LINEAR ? 1 : 2;
#pragma unroll
                        for (int c = 0; c < CHUNKS; ++c) {
                            float v[NOW][16];
                            tmem_load_rows16<NOW>(at + c * 16, TN, v, 0);
#pragma unroll
                            for (int a = 0; a < NOW; ++a)
#pragma unroll
                                for (int i = 0; i < 16; ++i) sum[c][a][i] += v[a][i];
                        }
                    }
                    give_back(b);
                    if (++b == SETS) { b = 0; phase ^= 1u; }
                }
                if (!ok) break;
#pragma unroll
                for (int c = 0; c < CHUNKS; ++c) {
                    if (split) put_share(c, sum[c][0]);
                    else finish<T, MODE>(p, q, row, col + c * 16, place_bias(c), sum[c]);
                }
            }
            if constexpr (MODE == LINEAR) {
                if (split) {  // the last share of this warp's part: all of them, in their order
                    __threadfence();
                    __syncwarp();
                    unsigned before = 0u;
                    if (lane == 0) before = atomicAdd(q.tickets + mine * EPILOGUE_WARPS + warp, 1u);
                    if (__shfl_sync(FULL, before, 0) + 1u == (unsigned)q.splits) {
                        __threadfence();
#pragma unroll
                        for (int c = 0; c < CHUNKS; ++c) {
                            float v[16];
#pragma unroll
                            for (int i = 0; i < 16; ++i) v[i] = 0.f;
#pragma unroll 2
                            for (int s = 0; s < q.splits; ++s) {
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    const float4 w = __ldcg(shares + s * per_share + (c * 4 + i) * 32);
                                    v[4 * i] += w.x; v[4 * i + 1] += w.y; v[4 * i + 2] += w.z; v[4 * i + 3] += w.w;
                                }
                            }
                            finish_linear<T>(q, row, col + c * 16, place_bias(c), v);
                        }
                    }
                }
            }
        }
    }
    fence_before();
    __syncthreads();
    if constexpr (PAIR) cluster_sync();
    fence_after();
    if (warp == EPILOGUE_WARPS) {
        if constexpr (PAIR) tmem_free_pair<S::TMEM>(tmem);
        else tmem_free<S::TMEM>(tmem);
    }
    if (threadIdx.x == 0) report_waits(gave_up, p.status);
}

}  // namespace tile
}  // namespace cf
