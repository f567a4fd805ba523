// The gated feed-forward of a few rows: the three weights are read once, which is all the time that it needs (at the largest sizes of
// a GPU's memory bandwidth, at the smallest of two launches in a chain).
//
// float32, and values that do not lie on 16 bytes: a group of `warps` warps computes UNITS neighbouring hidden units (then outputs) of
// all rows; lanes walk the contraction, four weights of each unit at a time, with the rows' values from L1.
//
// 16-bit types: multiplying and adding in float32 would take longer than the weights need to come (31 us for four rows of 2048 x 5632,
// whose 69 MB come in 10.6; 22 by what follows), so products are taken by mma.sync m16n8k16: 16 units by up to eight rows.  The sum does not mind which
// k an operand calls its own: lane t of a group of four takes eight neighbours, k = 8 t .. 8 t + 7 of each 32, of its two units and of
// its row, in one 16-byte load each, and both operands of two products are there.  A block's warps share the contraction.  The hidden
// units go from one kernel to the other as two values of the type, h and what its rounding left (1 us): 2^-22 of h in float16 and 2^-16
// in bfloat16 against the result's own rounding, 2^-11 and 2^-8 (float16: 2^-25 at least, half of its smallest number).
#pragma once
#include "common.cuh"
#include "tile_gemm.cuh"
#include "values.cuh"

namespace cf {

// Rows up to which this is taken, eight of mma.sync's columns; tiles take more.  us a call of 4, 8 rows here and of 9, 128 by tiles, one
// after the other in a graph:
//   128 x 512, float32        4.3, 6.4; 17.9, 19.6        bfloat16     4.0, 4.1; 12.4, 12.9
//   2048 x 5632, float32      38.5, 75.8; 142, 143        bfloat16     19.8, 21.0; 35.4, 34.4
//   2047 x 5631, bfloat16 (off 16 bytes)                               80.4, 74.2; 68.6, 66.2   (one row 36.3)
constexpr int GATED_ROWS = 8;

namespace rows {

constexpr int THREADS = 256;

template <int VEC>
__device__ __forceinline__ void load_hidden(const float *p, float (&v)[VEC])
{
    if constexpr (VEC == 1) {
        v[0] = *p;
    } else {
#pragma unroll
        for (int i = 0; i < VEC; i += 4) {
            const float4 w = *reinterpret_cast<const float4 *>(p + i);
            v[i] = w.x; v[i + 1] = w.y; v[i + 2] = w.z; v[i + 3] = w.w;
        }
    }
}

__device__ __forceinline__ float activation(int act, float g)
{
    return act == tile::SILU ? tile::gate_of<tile::SILU>(g).a : act == tile::GELU ? tile::gate_of<tile::GELU>(g).a : tile::gate_of<tile::RELU>(g).a;
}

// h (R, F): warp w of a group of `warps` takes every warps-th step of the contraction
template <class T, int VEC, int R, int UNITS>
__global__ void __launch_bounds__(THREADS) hidden_kernel(const __grid_constant__ cf_gated_ffn d, float *h, int warps)
{
    __shared__ float part[8][2 * UNITS * R];
    grid_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, in_group = warp % warps;
    const int unit0 = ((int)blockIdx.x * (8 / warps) + warp / warps) * UNITS, D = (int)d.D, F = (int)d.F;
    const T *x = static_cast<const T *>(d.x), *wg = static_cast<const T *>(d.w_gate), *wu = static_cast<const T *>(d.w_up);
    float g[UNITS][R], u[UNITS][R];
#pragma unroll
    for (int j = 0; j < UNITS; ++j)
#pragma unroll
        for (int r = 0; r < R; ++r) g[j][r] = u[j][r] = 0.f;
    grid_dependency_wait();
    for (int k = (in_group * 32 + lane) * VEC; k < D; k += warps * 32 * VEC) {
        float a[UNITS][VEC], b[UNITS][VEC];
#pragma unroll
        for (int j = 0; j < UNITS; ++j) {
            const long long at = (long long)min(unit0 + j, F - 1) * D + k;
            load_values<T, VEC>(wg + at, a[j]);
            load_values<T, VEC>(wu + at, b[j]);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float v[VEC];
            load_values<T, VEC>(x + (long long)min(r, (int)d.N - 1) * d.ldx + k, v);
#pragma unroll
            for (int j = 0; j < UNITS; ++j)
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    g[j][r] += a[j][e] * v[e];
                    u[j][r] += b[j][e] * v[e];
                }
        }
    }
#pragma unroll
    for (int j = 0; j < UNITS; ++j)
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float a = warp_sum(g[j][r]), b = warp_sum(u[j][r]);
            if (lane == 0) { part[warp][(j * R + r) * 2] = a; part[warp][(j * R + r) * 2 + 1] = b; }
        }
    __syncthreads();
    for (int i = in_group * 32 + lane; i < UNITS * R; i += warps * 32) {
        const int f = unit0 + i / R, r = i % R;
        if (f >= F || r >= d.N) continue;
        float a = 0.f, b = 0.f;
        for (int w = 0; w < warps; ++w) { a += part[warp - in_group + w][2 * i]; b += part[warp - in_group + w][2 * i + 1]; }
        if (d.b_gate) a += to_float(static_cast<const T *>(d.b_gate)[f]);
        if (d.b_up) b += to_float(static_cast<const T *>(d.b_up)[f]);
        h[(long long)r * F + f] = activation(d.activation, a) * b;
    }
}

template <class T, int VEC, int R, int UNITS>
__global__ void __launch_bounds__(THREADS) output_kernel(const __grid_constant__ cf_gated_ffn d, const float *h, T *y, int warps)
{
    __shared__ float part[8][UNITS * R];
    grid_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, in_group = warp % warps;
    const int unit0 = ((int)blockIdx.x * (8 / warps) + warp / warps) * UNITS, D = (int)d.D, F = (int)d.F;
    const T *wd = static_cast<const T *>(d.w_down);
    float s[UNITS][R];
#pragma unroll
    for (int j = 0; j < UNITS; ++j)
#pragma unroll
        for (int r = 0; r < R; ++r) s[j][r] = 0.f;
    const int stride = warps * 32 * VEC, k0 = (in_group * 32 + lane) * VEC;
    constexpr int AHEAD = 2;  // steps of weights on their way: the first ones from before the hidden units are there (they are the caller's)
    Raw<T, VEC> a[AHEAD][UNITS];
    auto fetch = [&](int t, int k) {
#pragma unroll
        for (int j = 0; j < UNITS; ++j) {
            a[t][j] = Raw<T, VEC>{};
            if (k < F) a[t][j] = load_raw<T, VEC>(wd + (long long)min(unit0 + j, D - 1) * F + k);
        }
    };
#pragma unroll
    for (int t = 0; t < AHEAD; ++t) fetch(t, k0 + t * stride);
    grid_dependency_wait();
    for (int k = k0; k < F; k += AHEAD * stride) {
#pragma unroll
        for (int t = 0; t < AHEAD; ++t) {
            const int at = k + t * stride;
            if (at >= F) break;
            float w[UNITS][VEC];
#pragma unroll
            for (int j = 0; j < UNITS; ++j) expand<T, VEC>(a[t][j], w[j]);
            fetch(t, at + AHEAD * stride);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float v[VEC];
                load_hidden<VEC>(h + (long long)min(r, (int)d.N - 1) * F + at, v);
#pragma unroll
                for (int j = 0; j < UNITS; ++j)
#pragma unroll
                    for (int e = 0; e < VEC; ++e) s[j][r] += w[j][e] * v[e];
            }
        }
    }
#pragma unroll
    for (int j = 0; j < UNITS; ++j)
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float a = warp_sum(s[j][r]);
            if (lane == 0) part[warp][j * R + r] = a;
        }
    __syncthreads();
    for (int i = in_group * 32 + lane; i < UNITS * R; i += warps * 32) {
        const int c = unit0 + i / R, r = i % R;
        if (c >= D || r >= d.N) continue;
        float a = 0.f;
        for (int w = 0; w < warps; ++w) a += part[warp - in_group + w][i];
        if (d.b_down) a += to_float(static_cast<const T *>(d.b_down)[c]);
        y[(long long)r * D + c] = from_float<T>(a);
    }
}

// Warps that share a group's contraction: while there are SMs without a block and steps to share.
inline int warps_of(long long units, int per_group, long long steps)
{
    int warps = 1;
    while (warps < 8 && steps > warps && (units + per_group - 1) / per_group * warps < 16ll * sm_count()) warps *= 2;
    return warps;
}

// ---- 16-bit types, on 16 bytes --------------------------------------------------------------------------------------------------
template <class T>
__device__ __forceinline__ void mma_16x8x16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    if constexpr (std::is_same<T, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 32 of the contraction: eight of them of units g and g + 8 (lo, hi) and of row g
template <class T>
__device__ __forceinline__ void mma_32(float (&c)[4], const uint4 &lo, const uint4 &hi, const uint4 &x)
{
    mma_16x8x16<T>(c, lo.x, hi.x, lo.y, hi.y, x.x, x.y);
    mma_16x8x16<T>(c, lo.z, hi.z, lo.w, hi.w, x.z, x.w);
}

// MATS matrices of (M, K) weights by up to eight rows x (ld) of K values: sums[mat][piece][unit of 16][row of 8] of the block's 16 units
// in `part`, (warps, MATS, PIECES, 16, 8).  MMA_AHEAD: steps of 32 on their way.  WAIT: x comes from the kernel before (the weights are
// the caller's, and are fetched earlier).  PIECES: x is the sum of so many matrices, `apart` values apart, whose sums are kept apart too.
template <class T, int MATS, int MMA_AHEAD, int PIECES, bool WAIT>
__device__ __forceinline__ void weigh_rows(const T *const (&w)[MATS], int M, int K, const T *x, long long ld, long long apart, int rows, int unit0, int warps,
                                           float *part)
{
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const long long lo = (long long)min(unit0 + g, M - 1) * K + 8 * t, hi = (long long)min(unit0 + g + 8, M - 1) * K + 8 * t;
    const T *xr = x + (long long)min(g, rows - 1) * ld + 8 * t;
    uint4 a[MMA_AHEAD][MATS][2];
    auto fetch = [&](int i, int k) {
#pragma unroll
        for (int m = 0; m < MATS; ++m) {
            a[i][m][0] = a[i][m][1] = make_uint4(0u, 0u, 0u, 0u);
            if (k + 8 * t < K) {
                a[i][m][0] = __ldg(reinterpret_cast<const uint4 *>(w[m] + lo + k));
                a[i][m][1] = __ldg(reinterpret_cast<const uint4 *>(w[m] + hi + k));
            }
        }
    };
    const int k0 = warp * 32, step = warps * 32;
#pragma unroll
    for (int i = 0; i < MMA_AHEAD; ++i) fetch(i, k0 + i * step);
    if constexpr (WAIT) grid_dependency_wait();
    float c[MATS][PIECES][4];
#pragma unroll
    for (int m = 0; m < MATS; ++m)
#pragma unroll
        for (int q = 0; q < PIECES; ++q)
#pragma unroll
            for (int i = 0; i < 4; ++i) c[m][q][i] = 0.f;
    for (int k = k0; k < K; k += MMA_AHEAD * step) {
        uint4 b[MMA_AHEAD][PIECES];
#pragma unroll
        for (int i = 0; i < MMA_AHEAD; ++i)
#pragma unroll
            for (int q = 0; q < PIECES; ++q) {
                const int at = k + i * step;
                b[i][q] = make_uint4(0u, 0u, 0u, 0u);
                if (at + 8 * t < K && g < rows) b[i][q] = *reinterpret_cast<const uint4 *>(xr + q * apart + at);
            }
#pragma unroll
        for (int i = 0; i < MMA_AHEAD; ++i) {
            const int at = k + i * step;
            if (at >= K) break;
#pragma unroll
            for (int m = 0; m < MATS; ++m)
#pragma unroll
                for (int q = 0; q < PIECES; ++q) mma_32<T>(c[m][q], a[i][m][0], a[i][m][1], b[i][q]);
            fetch(i, at + MMA_AHEAD * step);
        }
    }
#pragma unroll
    for (int m = 0; m < MATS; ++m)
#pragma unroll
        for (int q = 0; q < PIECES; ++q) {
            float *to = part + (((warp * MATS + m) * PIECES + q) * 16 + g) * 8 + 2 * t;
            to[0] = c[m][q][0]; to[1] = c[m][q][1];
            to[64] = c[m][q][2]; to[65] = c[m][q][3];
        }
    __syncthreads();
}

template <class T>
__global__ void __launch_bounds__(256, 3) hidden_mma_kernel(const __grid_constant__ cf_gated_ffn d, T *h)
{
    __shared__ float part[8 * 2 * 128];
    grid_launch_dependents();
    const int unit0 = blockIdx.x * 16, F = (int)d.F, N = (int)d.N;
    const T *const w[2] = {static_cast<const T *>(d.w_gate), static_cast<const T *>(d.w_up)};
    weigh_rows<T, 2, 3, 1, false>(w, F, (int)d.D, static_cast<const T *>(d.x), d.ldx, 0, N, unit0, 8, part);
    const int f = unit0 + (threadIdx.x & 15), r = threadIdx.x >> 4;
    if (r >= N || f >= F) return;
    float a = 0.f, b = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        a += part[(i * 2 * 16 + (threadIdx.x & 15)) * 8 + r];
        b += part[((i * 2 + 1) * 16 + (threadIdx.x & 15)) * 8 + r];
    }
    if (d.b_gate) a += to_float(static_cast<const T *>(d.b_gate)[f]);
    if (d.b_up) b += to_float(static_cast<const T *>(d.b_up)[f]);
    const float v = activation(d.activation, a) * b;
    // (the largest value stands for all beyond it, and what it leaves carries on: twice the range, then an infinity as by tiles)
    const float first = to_float(from_float<T>(v)), whole = fabsf(first) <= largest<T>() || first != first ? first : copysignf(largest<T>(), first);
    T *to = h + (long long)r * F + f;
    to[0] = from_float<T>(whole);
    to[(long long)N * F] = from_float<T>(v - whole);
}

template <class T>
__global__ void __launch_bounds__(512) output_mma_kernel(const __grid_constant__ cf_gated_ffn d, const T *h, T *y)
{
    __shared__ float part[16 * 2 * 128];
    grid_launch_dependents();
    const int unit0 = blockIdx.x * 16, D = (int)d.D, N = (int)d.N;
    const T *const w[1] = {static_cast<const T *>(d.w_down)};
    weigh_rows<T, 1, 6, 2, true>(w, D, (int)d.F, h, d.F, (long long)N * d.F, N, unit0, 16, part);
    const int c = unit0 + (threadIdx.x & 15), r = threadIdx.x >> 4;
    if (r >= N || c >= D) return;
    float a = 0.f, left = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        a += part[(i * 2 * 16 + (threadIdx.x & 15)) * 8 + r];
        left += part[((i * 2 + 1) * 16 + (threadIdx.x & 15)) * 8 + r];
    }
    if (fabsf(a) < INFINITY) a += left;  // (of an infinite weight what was left of h, zero or of the other sign, says nothing)
    if (d.b_down) a += to_float(static_cast<const T *>(d.b_down)[c]);
    y[(long long)r * D + c] = from_float<T>(a);
}

template <class T>
int launch_mma(const cf_gated_ffn &d, void *y, T *h, cudaStream_t s)
{
    hidden_mma_kernel<T><<<(unsigned)((d.F + 15) / 16), 256, 0, s>>>(d, h);
    launch_chained(output_mma_kernel<T>, dim3((unsigned)((d.D + 15) / 16)), dim3(512), 0, s, true, d, static_cast<const T *>(h), static_cast<T *>(y));
    return launch_status("gated_rows");
}

template <class T, int VEC_X, int VEC_H, int R>
int launch(const cf_gated_ffn &d, void *y, float *h, cudaStream_t s)
{
    constexpr int UNITS = 2, OUT_UNITS = 4;  // (outputs: a block reads all of h, from L2)
    const int hw = warps_of(d.F, UNITS, (d.D + 32 * VEC_X - 1) / (32 * VEC_X)), ow = warps_of(d.D, OUT_UNITS, (d.F + 32 * VEC_H - 1) / (32 * VEC_H));
    const long long hg = (d.F + UNITS - 1) / UNITS, og = (d.D + OUT_UNITS - 1) / OUT_UNITS;
    hidden_kernel<T, VEC_X, R, UNITS><<<(unsigned)((hg * hw + 7) / 8), THREADS, 0, s>>>(d, h, hw);
    launch_chained(output_kernel<T, VEC_H, R, OUT_UNITS>, dim3((unsigned)((og * ow + 7) / 8)), dim3(THREADS), 0, s, true, d, h, static_cast<T *>(y), ow);
    return launch_status("gated_rows");
}

}  // namespace rows

// y of up to GATED_ROWS rows; h: N F floats (or, by mma.sync, 2 N F values of the type).
template <class T>
int gated_rows(const cf_gated_ffn &d, void *y, float *h, cudaStream_t s)
{
    constexpr int V = 16 / sizeof(T);
    const bool wide = d.D % V == 0 && d.F % V == 0 && d.ldx % V == 0 && aligned_to(d.x, 16) && aligned_to(d.w_gate, 16) && aligned_to(d.w_up, 16) &&
                      aligned_to(d.w_down, 16);
    if constexpr (sizeof(T) == 2) {
        if (wide) return rows::launch_mma<T>(d, y, reinterpret_cast<T *>(h), s);
    }
    auto go = [&](auto rows) {
        constexpr int R = decltype(rows)::value;
        return sizeof(T) == 4 && wide ? rows::launch<T, sizeof(T) == 4 ? 4 : 1, sizeof(T) == 4 ? 4 : 1, R>(d, y, h, s) : rows::launch<T, 1, 1, R>(d, y, h, s);
    };
    if (d.N <= 1) return go(std::integral_constant<int, 1>());
    if (d.N <= 2) return go(std::integral_constant<int, 2>());
    if (d.N <= 4) return go(std::integral_constant<int, 4>());
    return go(std::integral_constant<int, 8>());
}

}  // namespace cf
