// Norms of the query and key heads with the rotation by positions, one pass forward and one backward.
//
//   r = 1 / sqrt(mean_d x_d^2 + eps),  y_d = w_d x_d r,
//   theta_p = 2 pi sum_c pos[n, c] wave[h, p, c],  (y_1, y_2) -> (y_1 cos - y_2 sin, y_1 sin + y_2 cos) for each of P pairs;
//   what lies behind the 2 P rotated entries of a head passes with its norm alone.
//   backward, g' = the output's gradient turned back:  gw_d = sum g'_d x_d r,  gx_d = r (w_d g'_d - x_d r^2 mean_d'(w g' x)).
//
// What a pass cannot do without is memory traffic (2 + 2 bytes or 4 + 4 a value forward), but heads are short and 16-bit values many:
// 58 to 64 % of the issue slots are taken at two blocks per SM, at 3.6 to 4.7 TB/s.  Neither is used up; each thread has one head on its
// way while it computes another, 16 KB on an SM in 16 bits, which is less than the bandwidth times the memory's latency.  So: an angle is computed once per key head and used
// for that key head and the query heads that share it.  A head is held by the fewest lanes (a power of two) that take it in slots of
// 2 VEC values - a pair of vectors whose entries are partners - so that sums of squares are a few shuffles and nothing is exchanged for
// the rotation.  A group of lanes walks the rows with the same heads of each: its weights stay in registers, and the next head's values
// are on their way while one is computed.  Key and query heads are separate code (with one loop over both, selects and predicates
// took half of the instructions: backward of 16,384 rows of 32 + 8 heads of 128, bfloat16, 167 us against 138).  16-byte vectors
// forward (72 us there, 101 with 8 bytes); backward 8 bytes, since 16 would need more registers than two blocks on an SM leave.
// Waves count cycles per unit of position: the products are exact (a rounded product and its fused remainder), whole turns are
// dropped before the parts are added, and an angle is off by 2^-24 turns out to 2^24 turns of an axis; whole-numbered waves on
// fractional coordinates thus do not see lattice translations at all.  133,120 rows of 8 + 8 heads of 16, float32, waves of each head:
// 65 us forward (4.2 TB/s), 91 us backward (4.5 TB/s).
//
// The weights' gradients are sums over all rows: each lane keeps its entries' in registers, a block adds its lanes' in a fixed order,
// and a second kernel adds the blocks'.
#include "common.cuh"
#include "values.cuh"

namespace cf {
namespace {

constexpr int THREADS = 256;

struct HeadArgs {
    cf_qk_norm d;
    const void *gq_out, *gk_out;  // backward: gradients of the outputs, (N, H, D) contiguous
    void *q_out, *k_out;          // outputs, or the inputs' gradients
    float *partial;               // (blocks, columns) sums of the weights' gradients: of wq, then of wk, each (1 or H, D)
    int columns, columns_q;
    int lanes;                    // of a head
    int slots;                    // of a head: 2 VEC values each
    int rotated;                  // slots of rotated values
    int units;                    // partitions of a token's heads: key head u and its queries; or, `single`, one head each
    int single;
};

struct Place {  // of a slot's two vectors in a head
    int a, b;
    bool has_b;
};

template <int VEC>
__device__ __forceinline__ Place place_of(const HeadArgs &p, int slot)
{
    if (slot < p.rotated && !p.d.interleaved) return {slot * VEC, (int)p.d.P + slot * VEC, true};
    return {slot * 2 * VEC, slot * 2 * VEC + VEC, slot * 2 * VEC + VEC < (int)p.d.D};  // (the rotated slots before it hold 2 P values)
}

__device__ __forceinline__ float lanes_sum(float v, int lanes)
{
    if (lanes > 1) v += __shfl_xor_sync(FULL, v, 1);
    if (lanes > 2) v += __shfl_xor_sync(FULL, v, 2);
    if (lanes > 4) v += __shfl_xor_sync(FULL, v, 4);
    if (lanes > 8) v += __shfl_xor_sync(FULL, v, 8);
    if (lanes > 16) v += __shfl_xor_sync(FULL, v, 16);
    return v;
}

// The pairs turned by their angles, or back.
template <bool INTERLEAVED, bool BACK, int SP, int VEC>
__device__ __forceinline__ void rotate(const float2 (&cs)[SP][VEC], float (&a)[SP][VEC], float (&b)[SP][VEC])
{
#pragma unroll
    for (int i = 0; i < SP; ++i) {
        if constexpr (INTERLEAVED && VEC > 1) {
#pragma unroll
            for (int e = 0; e < VEC; e += 2) {
                const float2 u = cs[i][e / 2], v = cs[i][VEC / 2 + e / 2];
                const float a0 = a[i][e], a1 = a[i][e + 1], b0 = b[i][e], b1 = b[i][e + 1];
                a[i][e] = BACK ? a0 * u.x + a1 * u.y : a0 * u.x - a1 * u.y;
                a[i][e + 1] = BACK ? a1 * u.x - a0 * u.y : a1 * u.x + a0 * u.y;
                b[i][e] = BACK ? b0 * v.x + b1 * v.y : b0 * v.x - b1 * v.y;
                b[i][e + 1] = BACK ? b1 * v.x - b0 * v.y : b1 * v.x + b0 * v.y;
            }
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float2 u = cs[i][e];
                const float x = a[i][e], y = b[i][e];
                a[i][e] = BACK ? x * u.x + y * u.y : x * u.x - y * u.y;
                b[i][e] = BACK ? y * u.x - x * u.y : y * u.x + x * u.y;
            }
        }
    }
}

// Cosines and sines of a lane's pairs at a row's position: exact products, whole turns dropped.  The waves come from L1 (that
// is 12 registers less than keeping them).
template <class T, int VEC, int SP, int C>
__device__ __forceinline__ void row_angles(const HeadArgs &p, const float *waves, int lane, const float (&pos)[3], float2 (&cs)[SP][VEC])
{
#pragma unroll
    for (int s = 0; s < SP; ++s) {
        const int slot = lane + s * p.lanes;
        if (slot >= p.rotated) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) cs[s][e] = make_float2(1.f, 0.f);
            continue;
        }
        float w[VEC * C];
        const float *at = waves + (long long)slot * VEC * C;
        if constexpr (VEC == 1) {
#pragma unroll
            for (int c = 0; c < C; ++c) w[c] = __ldg(at + c);
        } else {
#pragma unroll
            for (int i = 0; i < VEC * C / 4; ++i) {
                const float4 v = __ldg(reinterpret_cast<const float4 *>(at) + i);
                w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
            }
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            float whole = 0.f, rest = 0.f;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const float t = __fmul_rn(pos[c], w[e * C + c]);
                rest += __fmaf_rn(pos[c], w[e * C + c], -t);
                whole += t - rintf(t);
            }
            if constexpr (sizeof(T) == 2) {  // (the sine of the special functions: 2^-21 off, a thousandth of a 16-bit half step)
                whole += rest;
                whole -= rintf(whole);
                __sincosf(6.283185307179586f * whole, &cs[s][e].y, &cs[s][e].x);
            } else {
                sincospif(2.f * (whole + rest), &cs[s][e].y, &cs[s][e].x);
            }
        }
    }
}

// Forward and backward: groups of lanes walk the rows, each with one unit of every row's heads.
template <class T, int VEC, int SP, bool INTERLEAVED, bool BWD>
__global__ void __launch_bounds__(THREADS, SP > 1 ? 1 : 2) qk_norm_kernel(const HeadArgs p)
{
    using R = Raw<T, VEC>;
    extern __shared__ float shared[];
    const int lane = threadIdx.x & (p.lanes - 1), per_block = THREADS / p.lanes, D = (int)p.d.D, C = (int)p.d.C;
    const long long group = (long long)blockIdx.x * per_block + threadIdx.x / p.lanes, walk = (long long)gridDim.x * per_block / p.units;
    const bool walks = group < walk * p.units;  // (the last few of a grid that is no multiple of the units have none)
    const int u = (int)(group % p.units), shared_by = (int)(p.d.Hq / p.d.Hk);
    // heads of the unit: key head j, then its query heads; or (single) one head alone, which takes the queries' place
    const bool key_alone = p.single && u >= p.d.Hq;
    const int j = !p.single ? u : key_alone ? u - (int)p.d.Hq : u / shared_by;
    const int queries = p.single ? 1 : shared_by, q0 = p.single ? (key_alone ? j : u) : j * shared_by;

    bool on[SP], on_b[SP];
    int at_a[SP], to_b[SP];  // a slot's first vector in a head, and its second one from there
    const T *wq = static_cast<const T *>(key_alone ? p.d.wk : p.d.wq), *wk = static_cast<const T *>(p.d.wk);
    if (wq != nullptr) wq += (long long)q0 * (key_alone ? p.d.wk_head : p.d.wq_head);
    if (wk != nullptr) wk += (long long)j * p.d.wk_head;
    R wq_raw[SP][2], wk_raw[SP][2];  // the weights, as they lie in memory
#pragma unroll
    for (int i = 0; i < SP; ++i) {
        const int slot = lane + i * p.lanes;
        on[i] = slot < p.slots;
        const Place at = place_of<VEC>(p, on[i] ? slot : 0);
        on_b[i] = on[i] && at.has_b;
        at_a[i] = at.a;
        to_b[i] = at.b - at.a;
    }
    auto weights = [&](const T *w, R(&raw)[SP][2]) {
#pragma unroll
        for (int i = 0; i < SP; ++i) {
            raw[i][0] = raw[i][1] = R{};
            if (w != nullptr && on[i]) raw[i][0] = load_raw<T, VEC>(w + at_a[i]);
            if (w != nullptr && on_b[i]) raw[i][1] = load_raw<T, VEC>(w + at_a[i] + to_b[i]);
        }
    };
    weights(wq, wq_raw);
    weights(wk, wk_raw);
    const bool weighted_q = wq != nullptr, weighted_k = wk != nullptr;
    const float inv_d = 1.f / (float)D, eps = (float)p.d.eps;
    float sum_q[BWD ? SP : 1][2][VEC], sum_k[BWD ? SP : 1][2][VEC];
    if constexpr (BWD) {
#pragma unroll
        for (int i = 0; i < SP; ++i)
#pragma unroll
            for (int e = 0; e < VEC; ++e) sum_q[i][0][e] = sum_q[i][1][e] = sum_k[i][0][e] = sum_k[i][1][e] = 0.f;
    }
    // (all lanes of a warp make the same number of steps: those without a row repeat the last one and keep nothing)
    const int N = (int)p.d.N, row0 = walks ? (int)(group / p.units) : N, steps = walk > 0 ? (int)((N + walk - 1) / walk) : 0;
    auto row_of = [&](int step) { return (int)min(row0 + step * walk, (long long)N - 1); };
    // the unit's places in a row, of inputs and (contiguous) of outputs and their gradients
    const T *kx = static_cast<const T *>(p.d.k) + (long long)j * p.d.k_head;
    const T *qx = key_alone ? kx : static_cast<const T *>(p.d.q) + (long long)q0 * p.d.q_head;
    const int k_row = (int)p.d.k_row, q_row = key_alone ? k_row : (int)p.d.q_row, q_head = (int)p.d.q_head;
    const int k_out_row = (int)p.d.Hk * D, q_out_row = key_alone ? k_out_row : (int)p.d.Hq * D;
    const T *gk = static_cast<const T *>(p.gk_out) + j * D, *gq = key_alone ? gk : static_cast<const T *>(p.gq_out) + q0 * D;
    T *ky = static_cast<T *>(p.k_out) + j * D, *qy = key_alone ? ky : static_cast<T *>(p.q_out) + q0 * D;
    R xa[SP], xb[SP], ga[BWD ? SP : 1], gb[BWD ? SP : 1];
    auto fetch = [&](const T *x, const T *g) {
#pragma unroll
        for (int s = 0; s < SP; ++s) {
            xa[s] = xb[s] = R{};
            const T *from = x + at_a[s];
            if (on[s]) xa[s] = load_raw<T, VEC>(from);
            if (on_b[s]) xb[s] = load_raw<T, VEC>(from + to_b[s]);
            if constexpr (BWD) {
                ga[s] = gb[s] = R{};
                const T *gf = g + at_a[s];
                if (on[s]) ga[s] = load_raw<T, VEC>(gf);
                if (on_b[s]) gb[s] = load_raw<T, VEC>(gf + to_b[s]);
            }
        }
    };
    float pos[3] = {0.f, 0.f, 0.f};
    auto fetch_row = [&](int n) {
        if (p.single) fetch(qx + (long long)n * q_row, gq + (long long)n * q_out_row);
        else fetch(kx + (long long)n * k_row, gk + (long long)n * k_out_row);
        if (p.d.P > 0) {
            const float *from = p.d.pos + (long long)n * C;
            pos[0] = from[0];
            if (C > 1) pos[1] = from[1];
            if (C > 2) pos[2] = from[2];
        }
    };
    float2 cs[SP][VEC];
    float a[SP][VEC], b[SP][VEC], fa[BWD ? SP : 1][VEC], fb[BWD ? SP : 1][VEC];
    auto take = [&]() {
#pragma unroll
        for (int s = 0; s < SP; ++s) {
            expand<T, VEC>(xa[s], a[s]);
            expand<T, VEC>(xb[s], b[s]);
            if constexpr (BWD) {
                expand<T, VEC>(ga[s], fa[s]);
                expand<T, VEC>(gb[s], fb[s]);
            }
        }
    };
    // one head, taken: its norm, weights and rotation, or the gradients'
    auto head = [&](const R(&w)[SP][2], bool weighted, auto &sum, T *to, bool live) {
        float square = 0.f;
#pragma unroll
        for (int s = 0; s < SP; ++s)
#pragma unroll
            for (int e = 0; e < VEC; ++e) square += a[s][e] * a[s][e] + b[s][e] * b[s][e];
        if constexpr (BWD) rotate<INTERLEAVED, true>(cs, fa, fb);
        const float r = rsqrtf(lanes_sum(square, p.lanes) * inv_d + eps);
#pragma unroll
        for (int s = 0; s < SP; ++s)
#pragma unroll
            for (int e = 0; e < VEC; ++e) { a[s][e] *= r; b[s][e] *= r; }  // x r from here on
        if (weighted) {
#pragma unroll
            for (int s = 0; s < SP; ++s) {
                float wa[VEC], wb[VEC];
                expand<T, VEC>(w[s][0], wa);
                expand<T, VEC>(w[s][1], wb);
                if constexpr (!BWD) {
#pragma unroll
                    for (int e = 0; e < VEC; ++e) { a[s][e] *= wa[e]; b[s][e] *= wb[e]; }
                } else {
                    if (live) {  // (a value that is no number belongs to its own row's sums alone)
#pragma unroll
                        for (int e = 0; e < VEC; ++e) { sum[s][0][e] += fa[s][e] * a[s][e]; sum[s][1][e] += fb[s][e] * b[s][e]; }
                    }
#pragma unroll
                    for (int e = 0; e < VEC; ++e) { fa[s][e] *= wa[e]; fb[s][e] *= wb[e]; }
                }
            }
        }
        if constexpr (!BWD) {
            rotate<INTERLEAVED, false>(cs, a, b);
        } else {
            float dot = 0.f;
#pragma unroll
            for (int s = 0; s < SP; ++s)
#pragma unroll
                for (int e = 0; e < VEC; ++e) dot += a[s][e] * fa[s][e] + b[s][e] * fb[s][e];
            const float m = lanes_sum(dot, p.lanes) * inv_d;
#pragma unroll
            for (int s = 0; s < SP; ++s)
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    a[s][e] = r * (fa[s][e] - a[s][e] * m);
                    b[s][e] = r * (fb[s][e] - b[s][e] * m);
                }
        }
        if (live) {
#pragma unroll
            for (int s = 0; s < SP; ++s) {
                T *at = to + at_a[s];
                if (on[s]) store_values<T, VEC>(at, a[s]);
                if (on_b[s]) store_values<T, VEC>(at + to_b[s], b[s]);
            }
        }
    };
    const float *wave0 = p.d.waves + (p.d.wave_heads == 1 ? 0 : (long long)j) * p.d.P * C;
    if (steps > 0) fetch_row(row_of(0));
    for (int step = 0; step < steps; ++step) {
        const bool live = row0 + step * walk < N;
        const int n = row_of(step);
        if (C == 3) row_angles<T, VEC, SP, 3>(p, wave0, lane, pos, cs);
        else if (C == 2) row_angles<T, VEC, SP, 2>(p, wave0, lane, pos, cs);
        else row_angles<T, VEC, SP, 1>(p, wave0, lane, pos, cs);
        const T *x = qx + (long long)n * q_row;
        const long long out = (long long)n * q_out_row;
        const T *g = gq + out;
        T *y = qy + out;
        // a head's values are taken, the next one's fetched, then it is computed
        if (!p.single) {
            take();
            fetch(x, g);
            head(wk_raw, weighted_k, sum_k, ky + (long long)n * k_out_row, live);
        }
        for (int i = 0; i < queries; ++i) {
            take();
            if (i + 1 < queries) {
                x += q_head;
                g += D;
                fetch(x, g);
            } else if (step + 1 < steps) {
                fetch_row(row_of(step + 1));
            }
            head(wq_raw, weighted_q, sum_q, y, live);
            y += D;
        }
    }
    if constexpr (BWD) {
        if (p.partial == nullptr) return;
        const int first = (int)(((long long)blockIdx.x * per_block) % p.units);  // the block's first unit
        for (int which = 0; which < 2; ++which) {  // the queries' weights, the keys'
            const int begin = which ? p.columns_q : 0, end = which ? p.columns : p.columns_q;
            if (!(which && p.single)) {  // (single: all sums are in sum_q, and are there already)
                __syncthreads();
                float *mine = shared + (size_t)(threadIdx.x / p.lanes) * D;
#pragma unroll
                for (int s = 0; s < SP; ++s) {
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        if (on[s]) mine[at_a[s] + e] = which ? sum_k[s][0][e] : sum_q[s][0][e];
                        if (on_b[s]) mine[at_a[s] + to_b[s] + e] = which ? sum_k[s][1][e] : sum_q[s][1][e];
                    }
                }
                __syncthreads();
            }
            const bool each = end - begin > D;  // one set of sums per head (or there is one head)
            const int unit0 = p.single && which ? (int)p.d.Hq : 0, units = p.single ? (int)(which ? p.d.Hk : p.d.Hq) : p.units;
            for (int c = begin + threadIdx.x; c < end; c += THREADS) {
                const int set = (c - begin) / D, d = (c - begin) % D;
                float t = 0.f;
                if (each || units == 1) {
                    for (int g = (unit0 + set - first + p.units) % p.units; g < per_block; g += p.units) t += shared[(size_t)g * D + d];
                } else {
                    for (int g = 0; g < per_block; ++g) {
                        const int v = (first + g) % p.units - unit0;
                        if (v >= 0 && v < units) t += shared[(size_t)g * D + d];
                    }
                }
                p.partial[(size_t)blockIdx.x * p.columns + c] = t;
            }
        }
    }
}

// The blocks' sums, in a fixed order: 32 columns, a block's 32 warps a share of the blocks each.
template <class T>
__global__ void __launch_bounds__(1024) qk_weight_sum_kernel(const float *partial, int blocks, int columns, int columns_q, T *gwq, T *gwk)
{
    __shared__ float part[32][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    float t = 0.f;
    if (c < columns) {
#pragma unroll 8
        for (int b = warp; b < blocks; b += 32) t += partial[(size_t)b * columns + c];
    }
    part[warp][lane] = t;
    __syncthreads();
    if (warp > 0 || c >= columns) return;
#pragma unroll
    for (int w = 1; w < 32; ++w) t += part[w][lane];
    T *to = c < columns_q ? gwq : gwk;
    if (to != nullptr) to[c < columns_q ? c : c - columns_q] = from_float<T>(t);
}

// ---- host -----------------------------------------------------------------------------------------------------------------
int check_args(const char *who, const cf_qk_norm *d)
{
    CF_REQUIRE(d, CF_ERR_INVALID, "%s: null pointer", who);
    CF_REQUIRE(known_type(d->type), CF_ERR_UNSUPPORTED, "%s: type %d is none of CF_FLOAT32, CF_BFLOAT16, CF_FLOAT16", who, d->type);
    CF_REQUIRE(d->N >= 0 && d->Hq >= 1 && d->Hk >= 1 && d->D >= 1 && d->P >= 0 && d->C >= 0, CF_ERR_INVALID, "%s: negative size", who);
    CF_REQUIRE(d->D <= CF_QK_NORM_MAX_DIM && d->Hq <= 1024 && d->Hk <= 1024 && d->N < (1ll << 31) && d->N * (d->Hq + d->Hk) < (1ll << 31),
               CF_ERR_RANGE, "%s: N=%lld Hq=%lld Hk=%lld D=%lld", who, (long long)d->N, (long long)d->Hq, (long long)d->Hk, (long long)d->D);
    CF_REQUIRE(d->Hq % d->Hk == 0, CF_ERR_INVALID, "%s: %lld query heads do not share %lld key heads evenly", who, (long long)d->Hq, (long long)d->Hk);
    CF_REQUIRE(d->P <= d->D / 2, CF_ERR_INVALID, "%s: %lld pairs in heads of %lld", who, (long long)d->P, (long long)d->D);
    CF_REQUIRE(d->q_row < (1ll << 31) && d->q_head < (1ll << 31) && d->k_row < (1ll << 31) && d->k_head < (1ll << 31), CF_ERR_RANGE, "%s: stride of 2^31", who);
    CF_REQUIRE(d->q_row >= 0 && d->q_head >= 0 && d->k_row >= 0 && d->k_head >= 0, CF_ERR_INVALID, "%s: negative stride", who);
    CF_REQUIRE((d->wq_head == 0 || d->wq_head == d->D) && (d->wk_head == 0 || d->wk_head == d->D), CF_ERR_INVALID, "%s: weights are (D) or (H, D)", who);
    CF_REQUIRE(d->N == 0 || (d->q && d->k), CF_ERR_INVALID, "%s: null pointer", who);
    if (d->P > 0) {
        CF_REQUIRE(d->C >= 1 && d->C <= 3, CF_ERR_UNSUPPORTED, "%s: %lld position axes", who, (long long)d->C);
        CF_REQUIRE(d->wave_heads == 1 || d->wave_heads == d->Hk, CF_ERR_INVALID, "%s: waves of %lld heads for %lld key heads", who, (long long)d->wave_heads,
                   (long long)d->Hk);
        CF_REQUIRE(d->waves && (d->N == 0 || d->pos), CF_ERR_INVALID, "%s: null pointer", who);
    }
    return CF_OK;
}

// Whether all that is read and written lies on vectors of `vec` values, and the slots' borders too.
bool fits(const HeadArgs &a, int vec, bool backward)
{
    const cf_qk_norm &d = a.d;
    const size_t bytes = (size_t)vec * type_size(d.type);
    if (d.P % vec != 0 || (d.D - 2 * d.P) % (2 * vec) != 0) return false;
    for (long long st : {(long long)d.q_row, (long long)d.q_head, (long long)d.k_row, (long long)d.k_head})
        if (st % vec != 0) return false;
    if (!aligned_to(d.q, bytes) || !aligned_to(d.k, bytes) || !aligned_to(a.q_out, bytes) || !aligned_to(a.k_out, bytes) || !aligned_to(d.wq, bytes) ||
        !aligned_to(d.wk, bytes))
        return false;
    if (d.P > 0 && !aligned_to(d.waves, 16)) return false;
    return !backward || (aligned_to(a.gq_out, bytes) && aligned_to(a.gk_out, bytes));
}

constexpr int MAX_BLOCKS_PER_SM = 8;  // (2,048 threads)

// Blocks: `at_once` per SM walk the rows; no more groups than there are items, but every unit is walked.
long long blocks_of(long long items, int units, int per_block, int at_once)
{
    const long long cap = (long long)sm_count() * at_once, need = (items + per_block - 1) / per_block, least = (units + per_block - 1) / per_block;
    const long long blocks = need < cap ? need : cap;
    return blocks > least ? blocks : least;
}

int units_of(const cf_qk_norm &d, int &single)
{
    // query weights of each head, several query heads to a key head: one head per unit, so that a lane has one set of weights
    single = d.Hq != d.Hk && d.wq != nullptr && d.wq_head != 0;
    return (int)(single ? d.Hq + d.Hk : d.Hk);
}

template <class T, int VEC, int SP, bool INTERLEAVED, bool BWD>
int launch_sp(const HeadArgs &a, void *gwq, void *gwk, cudaStream_t s)
{
    static thread_local int resident[64] = {};
    const int per_block = THREADS / a.lanes;
    const size_t smem = BWD && a.partial ? (size_t)per_block * a.d.D * sizeof(float) : 0;
    int dev = 0;
    cudaGetDevice(&dev);
    int &at_once = resident[dev & 63];
    if (at_once == 0) {
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&at_once, qk_norm_kernel<T, VEC, SP, INTERLEAVED, BWD>, THREADS, 16384) != cudaSuccess || at_once < 1) {
            cudaGetLastError();
            at_once = 1;
        }
        if (at_once > MAX_BLOCKS_PER_SM) at_once = MAX_BLOCKS_PER_SM;
    }
    const long long blocks = blocks_of(a.d.N * a.units, a.units, per_block, at_once);
    qk_norm_kernel<T, VEC, SP, INTERLEAVED, BWD><<<(unsigned)blocks, THREADS, smem, s>>>(a);
    if (BWD && a.partial != nullptr)
        qk_weight_sum_kernel<T><<<(a.columns + 31) / 32, 1024, 0, s>>>(a.partial, (int)blocks, a.columns, a.columns_q, static_cast<T *>(gwq), static_cast<T *>(gwk));
    return launch_status("qk_norm_kernel");
}

template <class T, int VEC, bool INTERLEAVED, bool BWD>
int launch_vec(HeadArgs a, void *gwq, void *gwk, cudaStream_t s)
{
    a.rotated = (int)(a.d.P / VEC);
    a.slots = a.rotated + (int)((a.d.D - 2 * a.d.P + 2 * VEC - 1) / (2 * VEC));
    a.lanes = 1;
    while (a.lanes < 32 && a.lanes < a.slots) a.lanes *= 2;
    const int sp = (a.slots + a.lanes - 1) / a.lanes;
    if (sp <= 1) return launch_sp<T, VEC, 1, INTERLEAVED, BWD>(a, gwq, gwk, s);
    if constexpr (VEC <= 4) if (sp <= 2) return launch_sp<T, VEC, 2, INTERLEAVED, BWD>(a, gwq, gwk, s);  // (heads of up to 512: 64 slots of 8 values, 256 of 2)
    if constexpr (VEC == 1) return launch_sp<T, VEC, 8, INTERLEAVED, BWD>(a, gwq, gwk, s);
    return fail(CF_ERR_RANGE, "cf_qk_norm: heads of %lld", (long long)a.d.D);
}

template <class T, bool BWD>
int launch(const HeadArgs &a, void *gwq, void *gwk, cudaStream_t s)
{
    // (single values: pairs are taken one by one either way)
    if constexpr (sizeof(T) == 2 && !BWD) {
        if (fits(a, 8, BWD)) return a.d.interleaved ? launch_vec<T, 8, true, BWD>(a, gwq, gwk, s) : launch_vec<T, 8, false, BWD>(a, gwq, gwk, s);
    }
    if (fits(a, 4, BWD)) return a.d.interleaved ? launch_vec<T, 4, true, BWD>(a, gwq, gwk, s) : launch_vec<T, 4, false, BWD>(a, gwq, gwk, s);
    return launch_vec<T, 1, false, BWD>(a, gwq, gwk, s);
}

template <bool BWD>
int launch_typed(HeadArgs &a, void *gwq, void *gwk, void *stream)
{
    a.units = units_of(a.d, a.single);
    a.columns_q = a.d.wq ? (int)((a.d.wq_head ? a.d.Hq : 1) * a.d.D) : 0;
    a.columns = a.columns_q + (a.d.wk ? (int)((a.d.wk_head ? a.d.Hk : 1) * a.d.D) : 0);
    cudaStream_t s = as_stream(stream);
    if (a.d.type == CF_FLOAT32) return launch<float, BWD>(a, gwq, gwk, s);
    if (a.d.type == CF_BFLOAT16) return launch<__nv_bfloat16, BWD>(a, gwq, gwk, s);
    return launch<__half, BWD>(a, gwq, gwk, s);
}

}  // namespace
}  // namespace cf

using namespace cf;

extern "C" {

int cf_qk_norm_fwd(const cf_qk_norm *args, void *q_out, void *k_out, void *stream)
{
    const int rc = check_args("cf_qk_norm_fwd", args);
    if (rc != CF_OK) return rc;
    if (args->N == 0) return CF_OK;
    CF_REQUIRE(q_out && k_out, CF_ERR_INVALID, "cf_qk_norm_fwd: null pointer");
    HeadArgs a{};
    a.d = *args;
    a.q_out = q_out;
    a.k_out = k_out;
    return launch_typed<false>(a, nullptr, nullptr, stream);
}

int64_t cf_qk_norm_bwd_workspace_bytes(const cf_qk_norm *args)
{
    if (check_args("cf_qk_norm_bwd_workspace_bytes", args) != CF_OK) return 0;
    int single = 0;
    const int units = units_of(*args, single);
    // blocks of eight groups at least, as many as an SM holds at most: no launch of the call has more
    const long long blocks = blocks_of(args->N * units, units, THREADS / 32, MAX_BLOCKS_PER_SM);
    const long long columns = (args->wq ? (args->wq_head ? args->Hq : 1) : 0) + (args->wk ? (args->wk_head ? args->Hk : 1) : 0);
    return (int64_t)((size_t)blocks * columns * args->D * sizeof(float));
}

int cf_qk_norm_bwd(const cf_qk_norm *args, const void *gq_out, const void *gk_out, void *gq, void *gk, void *gwq, void *gwk, void *workspace, void *stream)
{
    const int rc = check_args("cf_qk_norm_bwd", args);
    if (rc != CF_OK) return rc;
    cudaStream_t s = as_stream(stream);
    const size_t size = type_size(args->type);
    CF_REQUIRE((gwq == nullptr || args->wq) && (gwk == nullptr || args->wk), CF_ERR_INVALID, "cf_qk_norm_bwd: the gradient of weights that are not there");
    if (args->N == 0) {
        if (gwq && cudaMemsetAsync(gwq, 0, (args->wq_head ? args->Hq : 1) * args->D * size, s) != cudaSuccess) return launch_status("cf_qk_norm_bwd");
        if (gwk && cudaMemsetAsync(gwk, 0, (args->wk_head ? args->Hk : 1) * args->D * size, s) != cudaSuccess) return launch_status("cf_qk_norm_bwd");
        return CF_OK;
    }
    CF_REQUIRE(gq_out && gk_out && gq && gk && ((!gwq && !gwk) || workspace), CF_ERR_INVALID, "cf_qk_norm_bwd: null pointer");
    CF_REQUIRE(aligned_to(workspace, 16), CF_ERR_INVALID, "cf_qk_norm_bwd: the workspace does not start on 16 bytes");
    HeadArgs a{};
    a.d = *args;
    a.gq_out = gq_out;
    a.gk_out = gk_out;
    a.q_out = gq;
    a.k_out = gk;
    a.partial = gwq || gwk ? static_cast<float *>(workspace) : nullptr;
    return launch_typed<true>(a, gwq, gwk, stream);
}

}  // extern "C"
