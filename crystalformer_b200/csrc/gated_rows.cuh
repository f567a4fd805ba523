// The gated feed-forward of a few rows: the three weights are read once, which is all the time that it needs (at the largest sizes of
// a GPU's memory bandwidth, at the smallest of two launches in a chain).  A group of WARPS warps computes UNITS neighbouring hidden
// units (then outputs) of all rows: lanes walk the contraction, eight or four weights of each unit at a time, with the rows' values
// from L1.  h stays float32 between the two kernels.
#pragma once
#include "common.cuh"
#include "tile_gemm.cuh"
#include "values.cuh"

namespace cf {

constexpr int GATED_ROWS = 8;  // rows up to which this pays against tiles of 128 rows

namespace rows {

constexpr int THREADS = 256;

template <class T, int VEC>
__device__ __forceinline__ void load_row(const T *p, int room, float (&v)[VEC])
{
    if constexpr (VEC > 1) {
        load_values<T, VEC>(p, v);
    } else {
        v[0] = room > 0 ? to_float(*p) : 0.f;
    }
}
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
    // two steps of weights on their way at a time
    const int stride = warps * 32 * VEC;
    for (int k = (in_group * 32 + lane) * VEC; k < D; k += 2 * stride) {
        Raw<T, VEC> a[2][UNITS], b[2][UNITS];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int j = 0; j < UNITS; ++j) {
                const long long at = (long long)min(unit0 + j, F - 1) * D + k + t * stride;
                a[t][j] = b[t][j] = Raw<T, VEC>{};
                if (k + t * stride < D) { a[t][j] = load_raw<T, VEC>(wg + at); b[t][j] = load_raw<T, VEC>(wu + at); }
            }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            if (k + t * stride >= D) break;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float v[VEC];
                load_values<T, VEC>(x + (long long)min(r, (int)d.N - 1) * d.ldx + k + t * stride, v);
#pragma unroll
                for (int j = 0; j < UNITS; ++j) {
                    float wa[VEC], wb[VEC];
                    expand<T, VEC>(a[t][j], wa);
                    expand<T, VEC>(b[t][j], wb);
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        g[j][r] += wa[e] * v[e];
                        u[j][r] += wb[e] * v[e];
                    }
                }
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
    while (warps < 8 && steps > warps && (units + per_group - 1) / per_group * warps < 24ll * sm_count()) warps *= 2;
    return warps;
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

// y of up to GATED_ROWS rows; h: N F floats.
template <class T>
int gated_rows(const cf_gated_ffn &d, void *y, float *h, cudaStream_t s)
{
    constexpr int V = 16 / sizeof(T);
    const bool wide = d.D % V == 0 && d.F % V == 0 && d.ldx % V == 0 && aligned_to(d.x, 16) && aligned_to(d.w_gate, 16) && aligned_to(d.w_up, 16) &&
                      aligned_to(d.w_down, 16);
    auto go = [&](auto rows) {
        constexpr int R = decltype(rows)::value;
        return wide ? rows::launch<T, V, V, R>(d, y, h, s) : rows::launch<T, 1, 1, R>(d, y, h, s);
    };
    if (d.N <= 1) return go(std::integral_constant<int, 1>());
    if (d.N <= 2) return go(std::integral_constant<int, 2>());
    if (d.N <= 4) return go(std::integral_constant<int, 4>());
    return go(std::integral_constant<int, 8>());
}

}  // namespace cf
