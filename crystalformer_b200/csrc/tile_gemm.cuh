// The tile products of the gated feed-forward on the fifth-generation tensor cores, in three modes:
//
//   LINEAR        C = A0 B0^T [+ A1 B1^T]                       epilogue: bias, stored in the type of the call; or float32 shares of a
//                                                               split contraction, which a second kernel adds
//   GLU_FORWARD   g = X Wg^T, u = X Wu^T                        epilogue: h = act(g + bg) (u + bu)
//   GLU_BACKWARD  the same, then dh = Gy Wd                     epilogue: h, dg = dh u act'(g), du = dh act(g)
//
// A block holds a 128 x TN tile of each accumulator in tensor memory and walks the contraction in blocks of 64: one thread keeps
// STAGES of them in flight by TMA (128-byte swizzle; either order of an operand, its contraction running along or across its rows), one
// thread issues tcgen05.mma, eight warps take the accumulators.  The grid is as large as the GPU and every block walks tiles, so
// that, with two sets of accumulators, a tile's epilogue runs beside the next one's products.
//
// 16-bit types: one product per pair of blocks; rows of 64 values are 128 bytes.  float32: an operand is the sum of three bfloat16
// pieces (24 bits, any exponent), made once by a packing kernel or by the epilogue that produces it, and a product is six: piece 0
// with 0, 1, 2, piece 1 with 0, 1 and piece 2 with 0 (what is left out is 2^-26 of a product).  The tensor core's running sums lose
// low bits with every instruction, so that with three pieces each block of 64 has accumulators of its own, smallest products first,
// and the sums over blocks are added in registers: errors are those of float32 sums (3e-7 relative at 512 terms).
//
// All waits are bounded (tc5::mbar_wait); one that runs out ends the block after its copies and products in flight.
#pragma once
#include <cuda.h>

#include "common.cuh"
#include "tc5.cuh"
#include "values.cuh"

namespace cf {
namespace tile {

enum Mode { LINEAR = 0, GLU_FORWARD = 1, GLU_BACKWARD = 2 };
enum Activation { SILU = 0, GELU = 1, RELU = 2 };

constexpr int TM = 128, TK = 64;
constexpr int EPILOGUE_WARPS = 8, THREADS = (EPILOGUE_WARPS + 2) * 32;

template <class T> constexpr int pieces_of = sizeof(T) == 4 ? 3 : 1;
template <class T> struct Piece { using type = T; };
template <> struct Piece<float> { using type = __nv_bfloat16; };

// Rows of pieces: value (row, col) of piece i at base + i * plane + row * ld + col.
struct Planes {
    void *base;
    long long ld, plane;
};

struct Params {
    CUtensorMap a[2], b[3];   // LINEAR: a[0] with b[0], a[1] with b[1]; GLU: a[0] with b[0] (gate) and b[1] (up), a[1] with b[2]
    int a_across[2], b_across[2];  // per part: the contraction runs across the rows of the operand
    int blocks0, blocks;      // of the contraction: of the first part, of both
    int m_tiles, n_tiles, splits;
    long long M;
    int N;
    // GLU
    const void *bias_gate, *bias_up;
    int act;
    Planes h, dg, du;
    int padded;               // columns that h, dg and du have memory for
    // LINEAR: rows [0, rows0) to out0, rows [row1, row1 + rows1) to out1
    void *out0, *out1;
    long long rows0, row1, rows1, ld_out;
    const void *bias;
    float *partial;           // (splits, M, N) instead
    unsigned *status;
};

template <class T, int MODE, int TN>
struct Shape {
    static constexpr int NP = pieces_of<T>;
    static constexpr int NB = MODE == LINEAR ? 1 : 2;                     // tiles of B per block of the contraction
    static constexpr int ACCS = MODE == LINEAR ? 1 : MODE == GLU_FORWARD ? 2 : 3;
    static constexpr int A_PIECE = TM * TK * 2, B_PIECE = NB * TN * TK * 2;
    static constexpr int STAGE = NP * (A_PIECE + B_PIECE);
    static constexpr int ROOM = 222 * 1024;
    static constexpr int STAGES = ROOM / STAGE < 8 ? ROOM / STAGE : 8;
    static constexpr int COLUMNS = ACCS * TN;                             // of one set of accumulators
    static constexpr int SETS = 2 * COLUMNS <= 512 ? 2 : 1;
    static constexpr int TMEM = SETS * COLUMNS <= 64 ? 64 : SETS * COLUMNS <= 128 ? 128 : SETS * COLUMNS <= 256 ? 256 : 512;
    static constexpr int MISC = STAGES * STAGE;
    static constexpr int SMEM = MISC + 256;
    static_assert(STAGES >= 2 && COLUMNS <= 512, "tile");
};

// ---- activations: value and derivative ---------------------------------------------------------------------------------------
struct Gate {
    float a, da;
};
template <int ACT>
__device__ __forceinline__ Gate gate_of(float g)
{
    if constexpr (ACT == SILU) {
        const float p = 1.f / (1.f + expf(-g));
        return {g * p, p * (1.f + g * (1.f - p))};
    } else if constexpr (ACT == GELU) {
        const float p = 0.5f * (1.f + erff(g * 0.70710678118654752f));
        return {g * p, p + g * expf(-0.5f * g * g) * 0.39894228040143268f};
    } else {
        // (a value that is no number stays one)
        return {g > 0.f || g != g ? g : 0.f, g > 0.f ? 1.f : 0.f};
    }
}

// The three bfloat16 pieces of two values, as words.
__device__ __forceinline__ void split_words(float a, float b, uint32_t (&w)[3])
{
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        w[i] = pack_two<__nv_bfloat16>(a, b);
        const float2 f = unpack_two<__nv_bfloat16>(w[i]);
        a -= f.x;
        b -= f.y;
    }
}

// 16 neighbours of a row into its planes; `room` columns from the first one on have memory (a multiple of eight).
template <class T>
__device__ __forceinline__ void store_planes(const Planes &to, long long row, int col, int room, const float (&v)[16])
{
    constexpr int NP = pieces_of<T>;
    using P = typename Piece<T>::type;
    P *at = static_cast<P *>(to.base) + row * to.ld + col;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        if (8 * half >= room) break;
        uint32_t w[NP][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float a = v[8 * half + 2 * i], b = v[8 * half + 2 * i + 1];
            if constexpr (NP == 3) {
                uint32_t s[3];
                split_words(a, b, s);
#pragma unroll
                for (int p = 0; p < 3; ++p) w[p][i] = s[p];
            } else {
                w[0][i] = pack_two<P>(a, b);
            }
        }
#pragma unroll
        for (int p = 0; p < NP; ++p) *reinterpret_cast<uint4 *>(at + p * to.plane + 8 * half) = make_uint4(w[p][0], w[p][1], w[p][2], w[p][3]);
    }
}

// 16 neighbours of a row of a matrix of any alignment; `room` of them exist.
template <class T>
__device__ __forceinline__ void store_run(T *to, int room, bool wide, const float (&v)[16])
{
    constexpr int VEC = 16 / sizeof(T);
    if (wide && room >= 16) {
#pragma unroll
        for (int i = 0; i < 16; i += VEC) {
            float w[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) w[e] = v[i + e];
            store_values<T, VEC>(to + i, w);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (i < room) to[i] = from_float<T>(v[i]);
    }
}

template <class T>
__device__ __forceinline__ void add_bias(const void *bias, int col, int room, float (&v)[16])
{
    if (bias == nullptr) return;
    const T *b = static_cast<const T *>(bias) + col;
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if (i < room) v[i] += to_float(b[i]);
}

// The epilogue of 16 columns of one row: v[acc][.] are the accumulators' values.
template <class T, int MODE, int ACT>
__device__ __forceinline__ void finish_glu(const Params &p, long long row, int col, float (&v)[MODE == GLU_FORWARD ? 2 : 3][16])
{
    const int room = p.N - col;
    add_bias<T>(p.bias_gate, col, room, v[0]);
    add_bias<T>(p.bias_up, col, room, v[1]);
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
    if (row >= p.M) return;
    store_planes<T>(p.h, row, col, p.padded - col, v[0]);
    if constexpr (MODE == GLU_BACKWARD) {
        store_planes<T>(p.du, row, col, p.padded - col, v[1]);
        store_planes<T>(p.dg, row, col, p.padded - col, v[2]);
    }
}

template <class T, int MODE, int COUNT>
__device__ __forceinline__ void finish(const Params &p, int split, long long row, int col, float (&v)[COUNT][16])
{
    if (col >= p.N) return;
    if constexpr (MODE == LINEAR) {
        if (row >= p.M) return;
        const int room = p.N - col;
        if (p.partial != nullptr) {
            store_run<float>(p.partial + ((long long)split * p.M + row) * p.N + col, room, (p.N & 3) == 0, v[0]);
            return;
        }
        add_bias<T>(p.bias, col, room, v[0]);
        T *to;
        if (row < p.rows0) to = static_cast<T *>(p.out0) + row * p.ld_out;
        else if (row >= p.row1 && row < p.row1 + p.rows1) to = static_cast<T *>(p.out1) + (row - p.row1) * p.ld_out;
        else return;
        store_run<T>(to + col, room, ((reinterpret_cast<uintptr_t>(to) & 15) | (p.ld_out & (16 / sizeof(T) - 1))) == 0, v[0]);
    } else {
        if (p.act == SILU) finish_glu<T, MODE, SILU>(p, row, col, v);
        else if (p.act == GELU) finish_glu<T, MODE, GELU>(p, row, col, v);
        else finish_glu<T, MODE, RELU>(p, row, col, v);
    }
}

struct Tile {
    int m, n, split;
    int k_lo, k_hi;
};
__device__ __forceinline__ Tile tile_of(const Params &p, long long t)
{
    // (columns run fastest: neighbours share rows of A, which are many, and the whole of B, which is small, stays in L2)
    Tile x;
    x.n = (int)(t % p.n_tiles);
    t /= p.n_tiles;
    x.m = (int)(t % p.m_tiles);
    x.split = (int)(t / p.m_tiles);
    x.k_lo = (int)((long long)p.blocks * x.split / p.splits);
    x.k_hi = (int)((long long)p.blocks * (x.split + 1) / p.splits);
    return x;
}

template <class T, int MODE, int TN>
__global__ void __launch_bounds__(THREADS, 1) tile_kernel(const __grid_constant__ Params p)
{
    using namespace tc5;
    using S = Shape<T, MODE, TN>;
    constexpr int NP = S::NP, STAGES = S::STAGES, SETS = S::SETS;
    extern __shared__ __align__(1024) unsigned char smem[];
    const uint32_t base = smem_u32(smem), misc = base + S::MISC;
    volatile unsigned *gave_up = reinterpret_cast<volatile unsigned *>(smem + S::MISC + 240);
    auto full = [&](int s) { return misc + 8u * (uint32_t)s; };
    auto empty = [&](int s) { return misc + 64u + 8u * (uint32_t)s; };
    auto ready = [&](int b) { return misc + 128u + 8u * (uint32_t)b; };
    auto taken = [&](int b) { return misc + 144u + 8u * (uint32_t)b; };
    const uint32_t drained = misc + 160u;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) { mbar_init(full(s), 1); mbar_init(empty(s), 1); }
        for (int b = 0; b < SETS; ++b) { mbar_init(ready(b), 1); mbar_init(taken(b), EPILOGUE_WARPS); }
        mbar_init(drained, 1);
        *gave_up = 0u;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_smem();
    }
    if (warp == EPILOGUE_WARPS) tmem_alloc<S::TMEM>(misc + 232);
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(smem + S::MISC + 232);
    grid_launch_dependents();
    grid_dependency_wait();
    const long long tiles = (long long)p.m_tiles * p.n_tiles * p.splits;

    if (warp == EPILOGUE_WARPS + 1) {
        // ---- copies ----
        if (lane == 0) {
            int s = 0;
            uint32_t phase = 1;
            bool ok = true;
            long long sent = 0;
            auto operand = [&](const CUtensorMap *map, bool across, uint32_t to, int rows, int row, int k, int piece, uint32_t bar) {
                if (!across) {
                    tma_load_3d(to, map, k, row, piece, bar);
                } else {
                    for (int i = 0; i < rows; i += 64) tma_load_3d(to + i * 128u, map, row + i, k, piece, bar);
                }
            };
            for (long long t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
                const Tile x = tile_of(p, t);
                for (int kb = x.k_lo; kb < x.k_hi; ++kb) {
                    ok = mbar_wait(empty(s), phase, gave_up);
                    if (!ok) break;
                    const int part = kb >= p.blocks0, k = (part ? kb - p.blocks0 : kb) * TK;
                    const uint32_t at = base + s * S::STAGE, bt = at + NP * S::A_PIECE;
                    const bool two = MODE != LINEAR && part == 0;  // gate and up
                    mbar_expect(full(s), (uint32_t)(NP * (S::A_PIECE + (two ? 2 : 1) * TN * TK * 2)));
#pragma unroll
                    for (int i = 0; i < NP; ++i) {
                        operand(&p.a[part], p.a_across[part], at + i * S::A_PIECE, TM, x.m * TM, k, i, full(s));
                        const uint32_t bi = bt + i * S::B_PIECE;
                        if (MODE == LINEAR) {
                            operand(&p.b[part], p.b_across[part], bi, TN, x.n * TN, k, i, full(s));
                        } else if (part == 0) {
                            operand(&p.b[0], p.b_across[0], bi, TN, x.n * TN, k, i, full(s));
                            operand(&p.b[1], p.b_across[0], bi + TN * TK * 2, TN, x.n * TN, k, i, full(s));
                        } else {
                            operand(&p.b[2], p.b_across[1], bi, TN, x.n * TN, k, i, full(s));
                        }
                    }
                    ++sent;
                    if (++s == STAGES) { s = 0; phase ^= 1u; }
                }
            }
            if (!ok) {  // the copies in flight land before the block goes: the last of each stage
                unsigned mine = 0u;
                for (int i = 0; i < STAGES && i < sent; ++i) {
                    if (--s < 0) { s = STAGES - 1; phase ^= 1u; }
                    mbar_wait(full(s), phase ^ 1u, &mine);
                }
            }
        }
    } else if (warp == EPILOGUE_WARPS) {
        // ---- products ----
        if (lane == 0) {
            constexpr int AB = sizeof(typename Piece<T>::type) == 2 && !std::is_same<typename Piece<T>::type, __half>::value ? 1 : 0;
            int s = 0, b = 0;
            uint32_t phase = 0, set_phase = 1;
            bool ok = true;
            for (long long t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
                const Tile x = tile_of(p, t);
                for (int kb = x.k_lo; kb < x.k_hi; ++kb) {
                    const bool fresh = NP > 1 || kb == x.k_lo;  // the first block of its accumulators
                    if (fresh) {
                        ok = mbar_wait(taken(b), set_phase, gave_up);
                        if (!ok) break;
                        fence_after();
                    }
                    ok = mbar_wait(full(s), phase, gave_up);
                    if (!ok) break;
                    fence_after();
                    const int part = kb >= p.blocks0;
                    const bool two = MODE != LINEAR && part == 0;
                    const uint32_t d = tmem + b * S::COLUMNS + (MODE == GLU_BACKWARD && part ? 2 * TN : 0);
                    const bool clear = fresh || (MODE == GLU_BACKWARD && kb == p.blocks0);
                    const bool aa = p.a_across[part], ba = p.b_across[part];
                    const uint32_t idesc = (two ? instr_desc<TM, 2 * TN <= 256 ? 2 * TN : 256, AB, false>() : instr_desc<TM, TN, AB, false>()) |
                                           (aa ? 1u << 15 : 0u) | (ba ? 1u << 16 : 0u);
                    // a step of 16 along the contraction: 32 bytes of a row, or 16 rows; panels of 64 across it lie 8 KB apart
                    const uint32_t a_step = (aa ? 2048 : 32) >> 4, b_step = (ba ? 2048 : 32) >> 4;
                    const uint32_t at = base + s * S::STAGE, bt = at + NP * S::A_PIECE;
                    const uint64_t a0 = smem_desc(at, 8192, 1024), b0 = smem_desc(bt, 8192, 1024);
                    constexpr uint32_t AP = S::A_PIECE >> 4, BP = S::B_PIECE >> 4;
                    if constexpr (NP == 1) {
#pragma unroll
                        for (int ks = 0; ks < TK / 16; ++ks) mma_f16(d, a0 + ks * a_step, b0 + ks * b_step, idesc, !(clear && ks == 0));
                    } else {
#pragma unroll
                        for (int ks = 0; ks < TK / 16; ++ks) {
                            const uint64_t ak = a0 + ks * a_step, bk = b0 + ks * b_step;
                            mma_f16(d, ak + 2 * AP, bk, idesc, ks > 0);
                            mma_f16(d, ak, bk + 2 * BP, idesc, true);
                            mma_f16(d, ak + AP, bk + BP, idesc, true);
                        }
#pragma unroll
                        for (int ks = 0; ks < TK / 16; ++ks) {
                            const uint64_t ak = a0 + ks * a_step, bk = b0 + ks * b_step;
                            mma_f16(d, ak + AP, bk, idesc, true);
                            mma_f16(d, ak, bk + BP, idesc, true);
                        }
#pragma unroll
                        for (int ks = 0; ks < TK / 16; ++ks) mma_f16(d, a0 + ks * a_step, b0 + ks * b_step, idesc, true);
                    }
                    mma_commit(empty(s));
                    if (++s == STAGES) { s = 0; phase ^= 1u; }
                    if (NP > 1 || kb == x.k_hi - 1) {
                        mma_commit(ready(b));
                        if (++b == SETS) { b = 0; set_phase ^= 1u; }
                    }
                }
            }
            if (!ok) {  // the instructions issued so far
                unsigned mine = 0u;
                mma_commit(drained);
                mbar_wait(drained, 0, &mine);
            }
        }
    } else {
        // ---- epilogue: warp w has rows 32 (w % 4) .. + 31 of the tile and half of its columns ----
        constexpr int CHUNKS = TN / 32;  // of 16 columns
        const int first = (warp >> 2) * (TN / 2);
        const uint32_t lanes = tmem + ((uint32_t)(warp & 3) << 21) + first;
        int b = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (long long t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
            const Tile x = tile_of(p, t);
            const long long row = (long long)x.m * TM + (warp & 3) * 32 + lane;
            const int col = x.n * TN + first;
            if constexpr (NP == 1) {
                ok = mbar_wait(ready(b), phase, gave_up);
                ok = __all_sync(FULL, ok);
                if (!ok) break;
                fence_after();
#pragma unroll
                for (int c = 0; c < CHUNKS; ++c) {
                    float v[S::ACCS][16];
                    tmem_load_rows16<S::ACCS>(lanes + b * S::COLUMNS + c * 16, TN, v);
                    if (c == CHUNKS - 1) {
                        fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(taken(b));
                    }
                    finish<T, MODE>(p, x.split, row, col + c * 16, v);
                }
                if (++b == SETS) { b = 0; phase ^= 1u; }
            } else {
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
                    const uint32_t at = lanes + b * S::COLUMNS;
                    if (MODE == GLU_BACKWARD && kb >= p.blocks0) {
#pragma unroll
                        for (int c = 0; c < CHUNKS; ++c) {
                            float v[1][16];
                            tmem_load_rows16<1>(at + 2 * TN + c * 16, TN, v);
#pragma unroll
                            for (int i = 0; i < 16; ++i) sum[c][S::ACCS - 1][i] += v[0][i];
                        }
                    } else {
                        constexpr int NOW = MODE == LINEAR ? 1 : 2;
#pragma unroll
                        for (int c = 0; c < CHUNKS; ++c) {
                            float v[NOW][16];
                            tmem_load_rows16<NOW>(at + c * 16, TN, v);
#pragma unroll
                            for (int a = 0; a < NOW; ++a)
#pragma unroll
                                for (int i = 0; i < 16; ++i) sum[c][a][i] += v[a][i];
                        }
                    }
                    fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(taken(b));
                    if (++b == SETS) { b = 0; phase ^= 1u; }
                }
                if (!ok) break;
#pragma unroll
                for (int c = 0; c < CHUNKS; ++c) finish<T, MODE>(p, x.split, row, col + c * 16, sum[c]);
            }
        }
    }
    fence_before();
    __syncthreads();
    fence_after();
    if (warp == EPILOGUE_WARPS) tmem_free<S::TMEM>(tmem);
    if (threadIdx.x == 0) report_waits(gave_up, p.status);
}

}  // namespace tile
}  // namespace cf
