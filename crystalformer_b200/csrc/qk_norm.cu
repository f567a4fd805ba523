// Norms of the query and key heads with the rotation by positions, one pass forward and one backward.
//
//   r = 1 / sqrt(mean_d x_d^2 + eps),  y_d = w_d x_d r,
//   theta_p = 2 pi sum_c pos[n, c] wave[h, p, c],  (y_1, y_2) -> (y_1 cos - y_2 sin, y_1 sin + y_2 cos) for each of P pairs;
//   what lies behind the 2 P rotated entries of a head passes with its norm alone.
//   backward, g' = the output's gradient turned back:  gw_d = sum g'_d x_d r,  gx_d = r (w_d g'_d - x_d r^2 mean_d'(w g' x)).
//
// Bound by memory (2 + 2 bytes or 4 + 4 a value forward), as long as the sines do not dominate: an angle is computed once per key
// head and used for that key head and the query heads that share it.  A head is held by the fewest lanes (a power of two) that
// take it in slots of 2 VEC values - a pair of vectors whose entries are partners - so that sums of squares are a few shuffles and
// nothing is exchanged for the rotation.  Waves count cycles per unit of position: the products are exact (a rounded product and
// its fused remainder), whole turns are dropped before the parts are added, and an angle is off by 2^-24 turns however far the
// position; whole-numbered waves on fractional coordinates thus do not see lattice translations at all.
//
// The weights' gradients are sums over all rows: each lane keeps its entries' in registers while it walks the rows, a block adds
// its lanes' in a fixed order, and a second kernel adds the blocks'.
#include "common.cuh"
#include "values.cuh"

namespace cf {
namespace {

constexpr int THREADS = 256;

struct HeadArgs {
    cf_qk_norm d;
    const void *gq_out, *gk_out;  // backward: gradients of the outputs, (N, H, D) contiguous
    void *q_out, *k_out;          // outputs, or the inputs' gradients
    float *partial;               // (blocks, units, D) sums of the weights' gradients
    int lanes;                    // of a head
    int slots;                    // of a head: 2 VEC values each
    int rotated;                  // slots of rotated values
    int units;                    // partitions of a token's heads: key head u and its queries; or, `single`, one head each
    int single;
};

template <int VEC>
struct Place {  // of a slot's two vectors in a head
    int a, b;
    bool has_b;
};

template <int VEC>
__device__ __forceinline__ Place<VEC> place_of(const HeadArgs &p, int slot)
{
    const int P = (int)p.d.P, D = (int)p.d.D;
    Place<VEC> at;
    if (slot < p.rotated && !p.d.interleaved) {
        at.a = slot * VEC;
        at.b = P + slot * VEC;
        at.has_b = true;
    } else {
        const int base = slot < p.rotated ? 0 : 2 * P - 2 * VEC * p.rotated;
        at.a = base + slot * 2 * VEC;
        at.b = at.a + VEC;
        at.has_b = at.b < D;
    }
    return at;
}

// cosine and sine of wave `pair` of key head j at a position, whole turns dropped
__device__ __forceinline__ float2 turn_of(const cf_qk_norm &d, const float (&pos)[3], long long j, int pair)
{
    const float *w = d.waves + ((d.wave_heads == 1 ? 0 : j) * d.P + pair) * d.C;
    float whole = 0.f, rest = 0.f;
#pragma unroll
    for (int c = 0; c < 3; ++c) {
        if (c >= d.C) break;
        const float t = __fmul_rn(pos[c], w[c]), e = __fmaf_rn(pos[c], w[c], -t);
        whole += t - rintf(t);
        rest += e - rintf(e);
    }
    whole -= rintf(whole);
    float2 cs;
    sincospif(2.f * (whole + rest), &cs.y, &cs.x);
    return cs;
}

// The slots of one lane: SP of them, `lanes` apart.
template <class T, int VEC, int SP>
struct Lane {
    Place<VEC> at[SP];
    bool on[SP];
    float2 cs[SP][VEC];

    __device__ __forceinline__ void init(const HeadArgs &p, int lane)
    {
#pragma unroll
        for (int i = 0; i < SP; ++i) {
            const int slot = lane + i * p.lanes;
            on[i] = slot < p.slots;
            at[i] = place_of<VEC>(p, on[i] ? slot : 0);
        }
    }
    __device__ __forceinline__ void turn(const HeadArgs &p, int lane, const float (&pos)[3], long long j)
    {
#pragma unroll
        for (int i = 0; i < SP; ++i) {
            const int slot = lane + i * p.lanes;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                cs[i][e] = make_float2(1.f, 0.f);
                if (on[i] && slot < p.rotated) cs[i][e] = turn_of(p.d, pos, j, slot * VEC + e);
            }
        }
    }
    __device__ __forceinline__ void load(const T *x, float (&a)[SP][VEC], float (&b)[SP][VEC]) const
    {
#pragma unroll
        for (int i = 0; i < SP; ++i) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) a[i][e] = b[i][e] = 0.f;
            if (on[i]) {
                load_values<T, VEC>(x + at[i].a, a[i]);
                if (at[i].has_b) load_values<T, VEC>(x + at[i].b, b[i]);
            }
        }
    }
    __device__ __forceinline__ void store(T *x, const float (&a)[SP][VEC], const float (&b)[SP][VEC]) const
    {
#pragma unroll
        for (int i = 0; i < SP; ++i) {
            if (on[i]) {
                store_values<T, VEC>(x + at[i].a, a[i]);
                if (at[i].has_b) store_values<T, VEC>(x + at[i].b, b[i]);
            }
        }
    }
    // the pairs turned by their angles (sign 1) or back (-1)
    __device__ __forceinline__ void rotate(bool interleaved, float sign, float (&a)[SP][VEC], float (&b)[SP][VEC]) const
    {
#pragma unroll
        for (int i = 0; i < SP; ++i) {
            if (interleaved && VEC > 1) {
#pragma unroll
                for (int e = 0; e < VEC; e += 2) {
                    const float2 u = cs[i][e / 2], v = cs[i][VEC / 2 + e / 2];
                    const float a0 = a[i][e], a1 = a[i][e + 1], b0 = b[i][e], b1 = b[i][e + 1];
                    a[i][e] = a0 * u.x - sign * a1 * u.y;
                    a[i][e + 1] = a1 * u.x + sign * a0 * u.y;
                    b[i][e] = b0 * v.x - sign * b1 * v.y;
                    b[i][e + 1] = b1 * v.x + sign * b0 * v.y;
                }
            } else {
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float2 u = cs[i][e];
                    const float x = a[i][e], y = b[i][e];
                    a[i][e] = x * u.x - sign * y * u.y;
                    b[i][e] = y * u.x + sign * x * u.y;
                }
            }
        }
    }
};

__device__ __forceinline__ float lanes_sum(float v, int lanes)
{
    for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
    return v;
}

template <int SP, int VEC>
__device__ __forceinline__ float dot_of(const float (&a)[SP][VEC], const float (&b)[SP][VEC], const float (&c)[SP][VEC], const float (&d)[SP][VEC])
{
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < SP; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) t += a[i][e] * c[i][e] + b[i][e] * d[i][e];
    return t;
}

__device__ __forceinline__ void position_of(const cf_qk_norm &d, long long n, float (&pos)[3])
{
#pragma unroll
    for (int c = 0; c < 3; ++c) pos[c] = d.P > 0 && c < d.C ? d.pos[n * d.C + c] : 0.f;
}

// Which heads unit u of a token has: key head `key` (or none), query heads [lo, hi); j: the key head whose waves they use.
struct Unit {
    long long key, lo, hi, j;
};
__device__ __forceinline__ Unit unit_of(const HeadArgs &p, int u)
{
    const long long group = p.d.Hk > 0 ? p.d.Hq / p.d.Hk : 1;
    if (!p.single) return {u, u * group, (u + 1) * group, u};
    if (u < p.d.Hq) return {-1, u, u + 1, u / group};
    return {u - p.d.Hq, 0, 0, u - p.d.Hq};
}

template <class T, int VEC, int SP>
__global__ void __launch_bounds__(THREADS) qk_norm_fwd_kernel(const HeadArgs p)
{
    const int lane = threadIdx.x & (p.lanes - 1), per_block = THREADS / p.lanes;
    const long long item = (long long)blockIdx.x * per_block + threadIdx.x / p.lanes, items = p.d.N * p.units;
    // (lanes of a warp beyond the last item go along for the shuffles, with the last one's values, and store nothing)
    const bool live = item < items;
    const long long at = live ? item : items - 1, n = at / p.units;
    const Unit unit = unit_of(p, (int)(at % p.units));
    Lane<T, VEC, SP> me;
    me.init(p, lane);
    float pos[3];
    position_of(p.d, n, pos);
    me.turn(p, lane, pos, unit.j);
    const float inv_d = 1.f / (float)p.d.D, eps = (float)p.d.eps;
    auto head = [&](const T *x, const T *w, T *to) {
        float a[SP][VEC], b[SP][VEC];
        me.load(x, a, b);
        const float r = rsqrtf(lanes_sum(dot_of(a, b, a, b), p.lanes) * inv_d + eps);
        if (w != nullptr) {
            float wa[SP][VEC], wb[SP][VEC];
            me.load(w, wa, wb);
#pragma unroll
            for (int i = 0; i < SP; ++i)
#pragma unroll
                for (int e = 0; e < VEC; ++e) { a[i][e] *= r * wa[i][e]; b[i][e] *= r * wb[i][e]; }
        } else {
#pragma unroll
            for (int i = 0; i < SP; ++i)
#pragma unroll
                for (int e = 0; e < VEC; ++e) { a[i][e] *= r; b[i][e] *= r; }
        }
        me.rotate(p.d.interleaved, 1.f, a, b);
        if (live) me.store(to, a, b);
    };
    const T *wq = static_cast<const T *>(p.d.wq), *wk = static_cast<const T *>(p.d.wk);
    if (unit.key >= 0)
        head(static_cast<const T *>(p.d.k) + n * p.d.k_row + unit.key * p.d.k_head, wk == nullptr ? wk : wk + unit.key * p.d.wk_head,
             static_cast<T *>(p.k_out) + (n * p.d.Hk + unit.key) * p.d.D);
    for (long long h = unit.lo; h < unit.hi; ++h)
        head(static_cast<const T *>(p.d.q) + n * p.d.q_row + h * p.d.q_head, wq == nullptr ? wq : wq + h * p.d.wq_head,
             static_cast<T *>(p.q_out) + (n * p.d.Hq + h) * p.d.D);
}

// A lane keeps the sums of its entries' weight gradients for queries and for keys: every unit of a lane's walk is the same one,
// which has one query head, or weights that its query heads share.
template <class T, int VEC, int SP>
__global__ void __launch_bounds__(THREADS) qk_norm_bwd_kernel(const HeadArgs p)
{
    extern __shared__ float shared[];
    const int lane = threadIdx.x & (p.lanes - 1), per_block = THREADS / p.lanes;
    const long long group = (long long)blockIdx.x * per_block + threadIdx.x / p.lanes, walk = (long long)gridDim.x * per_block / p.units;
    const bool walks = group < walk * p.units;  // (the last few of a grid that is no multiple of the units have none)
    const int u = (int)(group % p.units);
    const Unit unit = unit_of(p, u);
    Lane<T, VEC, SP> me;
    me.init(p, lane);
    const float inv_d = 1.f / (float)p.d.D, eps = (float)p.d.eps;
    float sum_q[2][SP][VEC], sum_k[2][SP][VEC];
#pragma unroll
    for (int i = 0; i < SP; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) sum_q[0][i][e] = sum_q[1][i][e] = sum_k[0][i][e] = sum_k[1][i][e] = 0.f;
    auto head = [&](const T *x, const T *w, const T *gout, T *to, bool live, float (&sum)[2][SP][VEC]) {
        float a[SP][VEC], b[SP][VEC], ga[SP][VEC], gb[SP][VEC];
        me.load(x, a, b);
        me.load(gout, ga, gb);
        me.rotate(p.d.interleaved, -1.f, ga, gb);
        const float r = rsqrtf(lanes_sum(dot_of(a, b, a, b), p.lanes) * inv_d + eps);
        if (w != nullptr) {
            float wa[SP][VEC], wb[SP][VEC];
            me.load(w, wa, wb);
            const float rl = live ? r : 0.f;
#pragma unroll
            for (int i = 0; i < SP; ++i)
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    if (live) {  // (a value that is no number belongs to its own row's sums alone)
                        sum[0][i][e] += ga[i][e] * (a[i][e] * rl);
                        sum[1][i][e] += gb[i][e] * (b[i][e] * rl);
                    }
                    ga[i][e] *= wa[i][e];
                    gb[i][e] *= wb[i][e];
                }
        }
        const float m = lanes_sum(dot_of(a, b, ga, gb), p.lanes) * inv_d * r * r;
#pragma unroll
        for (int i = 0; i < SP; ++i)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                a[i][e] = r * (ga[i][e] - a[i][e] * m);
                b[i][e] = r * (gb[i][e] - b[i][e] * m);
            }
        if (live) me.store(to, a, b);
    };
    const T *wq = static_cast<const T *>(p.d.wq), *wk = static_cast<const T *>(p.d.wk);
    // (all lanes of a warp make the same number of steps: those without a row repeat the last one and keep nothing)
    const long long steps = walk > 0 ? (p.d.N + walk - 1) / walk : 0;
    for (long long step = 0; step < steps; ++step) {
        const long long row = group / p.units + step * walk;
        const bool live = walks && row < p.d.N;
        const long long n = live ? row : p.d.N - 1;
        float pos[3];
        position_of(p.d, n, pos);
        me.turn(p, lane, pos, unit.j);
        auto query = [&](long long h) {
            head(static_cast<const T *>(p.d.q) + n * p.d.q_row + h * p.d.q_head, wq == nullptr ? wq : wq + h * p.d.wq_head,
                 static_cast<const T *>(p.gq_out) + (n * p.d.Hq + h) * p.d.D, static_cast<T *>(p.q_out) + (n * p.d.Hq + h) * p.d.D, live, sum_q);
        };
        if (!p.single) {
            head(static_cast<const T *>(p.d.k) + n * p.d.k_row + unit.j * p.d.k_head, wk == nullptr ? wk : wk + unit.j * p.d.wk_head,
                 static_cast<const T *>(p.gk_out) + (n * p.d.Hk + unit.j) * p.d.D, static_cast<T *>(p.k_out) + (n * p.d.Hk + unit.j) * p.d.D, live, sum_k);
            for (long long h = unit.lo; h < unit.hi; ++h) query(h);
        } else {  // (the heads of a warp's lanes differ: one call for either kind, as they shuffle together)
            const bool is_key = unit.key >= 0;
            const long long h = is_key ? unit.key : unit.lo, H = is_key ? p.d.Hk : p.d.Hq;
            const T *x = static_cast<const T *>(is_key ? p.d.k : p.d.q) + n * (is_key ? p.d.k_row : p.d.q_row) + h * (is_key ? p.d.k_head : p.d.q_head);
            const T *w = is_key ? (wk == nullptr ? wk : wk + h * p.d.wk_head) : wq + h * p.d.wq_head;
            const long long at = (n * H + h) * p.d.D;
            head(x, w, static_cast<const T *>(is_key ? p.gk_out : p.gq_out) + at, static_cast<T *>(is_key ? p.k_out : p.q_out) + at, live, sum_q);
        }
    }
    if (p.partial == nullptr) return;
    // (block, query or key, unit, entry)
    const int D = (int)p.d.D;
    for (int which = 0; which < (p.single ? 1 : 2); ++which) {  // (single: the unit says which)
        float(&sum)[2][SP][VEC] = which ? sum_k : sum_q;
        __syncthreads();
        float *mine = shared + (size_t)(threadIdx.x / p.lanes) * D;
#pragma unroll
        for (int i = 0; i < SP; ++i) {
            if (!me.on[i]) continue;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                mine[me.at[i].a + e] = sum[0][i][e];
                if (me.at[i].has_b) mine[me.at[i].b + e] = sum[1][i][e];
            }
        }
        __syncthreads();
        float *to = p.partial + ((size_t)blockIdx.x * 2 + which) * p.units * D;
        const int first = (int)(((long long)blockIdx.x * per_block) % p.units);  // the block's first unit
        for (int at = threadIdx.x; at < p.units * D; at += THREADS) {
            const int v = at / D, d = at % D;
            float t = 0.f;
            for (int g = (v - first + p.units) % p.units; g < per_block; g += p.units) t += shared[(size_t)g * D + d];
            to[at] = t;
        }
    }
}

// The blocks' sums, in their order: thread (x, y) column x of a unit's entry, the y-th share of the blocks.
template <class T>
__global__ void __launch_bounds__(256) qk_weight_sum_kernel(const HeadArgs p, int blocks, T *gwq, T *gwk)
{
    __shared__ float part[8][32];
    const int which = blockIdx.y, D = (int)p.d.D, lane = threadIdx.x & 31, share = threadIdx.x >> 5;
    T *to = which ? gwk : gwq;
    if (to == nullptr) return;
    const long long heads = which ? p.d.Hk : p.d.Hq;
    const bool each = (which ? p.d.wk_head : p.d.wq_head) != 0;
    // outputs: (heads, D), or (D) summed over the units
    const long long outs = each ? heads * D : D, at = (long long)blockIdx.x * 32 + lane;
    float t = 0.f;
    if (at < outs) {
        const int d = (int)(at % D);
        const long long h = at / D;
        // the units that hold it: of shared weights all; else the one of this head
        const long long u0 = (p.single && which ? p.d.Hq : 0) + (each ? h : 0), u1 = each ? u0 + 1 : p.units;
        for (int b = share; b < blocks; b += 8)
            for (long long u = u0; u < u1; ++u) t += p.partial[(((size_t)b * 2 + (p.single ? 0 : which)) * p.units + u) * D + d];
    }
    part[share][lane] = t;
    __syncthreads();
    if (share == 0 && at < outs) {
#pragma unroll
        for (int s = 1; s < 8; ++s) t += part[s][lane];
        to[at] = from_float<T>(t);
    }
}

// ---- host -----------------------------------------------------------------------------------------------------------------
int check_args(const char *who, const cf_qk_norm *d)
{
    CF_REQUIRE(d, CF_ERR_INVALID, "%s: null pointer", who);
    CF_REQUIRE(known_type(d->type), CF_ERR_UNSUPPORTED, "%s: type %d is none of CF_FLOAT32, CF_BFLOAT16, CF_FLOAT16", who, d->type);
    CF_REQUIRE(d->N >= 0 && d->Hq >= 1 && d->Hk >= 1 && d->D >= 1 && d->P >= 0 && d->C >= 0, CF_ERR_INVALID, "%s: negative size", who);
    CF_REQUIRE(d->D <= CF_QK_NORM_MAX_DIM && d->Hq <= 1024 && d->N * (d->Hq + d->Hk) < (1ll << 31), CF_ERR_RANGE, "%s: N=%lld Hq=%lld Hk=%lld D=%lld",
               who, (long long)d->N, (long long)d->Hq, (long long)d->Hk, (long long)d->D);
    CF_REQUIRE(d->Hq % d->Hk == 0, CF_ERR_INVALID, "%s: %lld query heads do not share %lld key heads evenly", who, (long long)d->Hq, (long long)d->Hk);
    CF_REQUIRE(2 * d->P <= d->D, CF_ERR_INVALID, "%s: %lld pairs in heads of %lld", who, (long long)d->P, (long long)d->D);
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
    return !backward || (aligned_to(a.gq_out, bytes) && aligned_to(a.gk_out, bytes));
}

constexpr int BWD_BLOCKS_PER_SM = 6;

long long bwd_blocks(long long items, int per_block)  // (no more groups than there are items)
{
    const long long cap = (long long)sm_count() * BWD_BLOCKS_PER_SM, need = (items + per_block - 1) / per_block;
    return need < cap ? need : cap;
}

int units_of(const cf_qk_norm &d, bool backward, int &single)
{
    // per-head query weights with several query heads to a key head: one head per unit, so that a lane has one set of sums
    single = backward && d.Hq != d.Hk && d.wq != nullptr && d.wq_head != 0;
    return (int)(single ? d.Hq + d.Hk : d.Hk);
}

template <class T, int VEC, int SP>
int launch_sp(const HeadArgs &a, bool backward, void *gwq, void *gwk, cudaStream_t s)
{
    const int per_block = THREADS / a.lanes;
    const long long items = a.d.N * a.units;
    if (!backward) {
        qk_norm_fwd_kernel<T, VEC, SP><<<(unsigned)((items + per_block - 1) / per_block), THREADS, 0, s>>>(a);
        return launch_status("qk_norm_fwd_kernel");
    }
    long long blocks = bwd_blocks(items, per_block);
    if (blocks * per_block < a.units) blocks = (a.units + per_block - 1) / per_block;  // (every unit is walked)
    const size_t smem = a.partial ? (size_t)per_block * a.d.D * sizeof(float) : 0;
    qk_norm_bwd_kernel<T, VEC, SP><<<(unsigned)blocks, THREADS, smem, s>>>(a);
    if (a.partial != nullptr) {
        const long long outs = (a.d.wq_head || a.d.wk_head ? a.d.Hq : 1) * a.d.D;
        qk_weight_sum_kernel<T><<<dim3((unsigned)((outs + 31) / 32), 2), 256, 0, s>>>(a, (int)blocks, static_cast<T *>(gwq), static_cast<T *>(gwk));
    }
    return launch_status("qk_norm_bwd_kernel");
}

template <class T, int VEC>
int launch_vec(HeadArgs a, bool backward, void *gwq, void *gwk, cudaStream_t s)
{
    a.rotated = (int)(a.d.P / VEC);
    a.slots = a.rotated + (int)((a.d.D - 2 * a.d.P + 2 * VEC - 1) / (2 * VEC));
    a.lanes = 1;
    while (a.lanes < 32 && a.lanes < a.slots) a.lanes *= 2;
    const int sp = (a.slots + a.lanes - 1) / a.lanes;
    if (sp <= 1) return launch_sp<T, VEC, 1>(a, backward, gwq, gwk, s);
    if constexpr (VEC <= 4) {  // (heads of up to 512: 32 slots of 16 values, 64 of 8, 256 of 2)
        if (sp <= 2) return launch_sp<T, VEC, 2>(a, backward, gwq, gwk, s);
    }
    if constexpr (VEC == 1) return launch_sp<T, VEC, 8>(a, backward, gwq, gwk, s);
    return fail(CF_ERR_RANGE, "cf_qk_norm: heads of %lld", (long long)a.d.D);
}

template <class T>
int launch(const HeadArgs &a, bool backward, void *gwq, void *gwk, cudaStream_t s)
{
    if constexpr (sizeof(T) == 2) {
        if (fits(a, 8, backward)) return launch_vec<T, 8>(a, backward, gwq, gwk, s);
    }
    if (fits(a, 4, backward)) return launch_vec<T, 4>(a, backward, gwq, gwk, s);
    return launch_vec<T, 1>(a, backward, gwq, gwk, s);
}

int launch_typed(HeadArgs &a, bool backward, void *gwq, void *gwk, void *stream)
{
    a.units = units_of(a.d, backward, a.single);
    cudaStream_t s = as_stream(stream);
    if (a.d.type == CF_FLOAT32) return launch<float>(a, backward, gwq, gwk, s);
    if (a.d.type == CF_BFLOAT16) return launch<__nv_bfloat16>(a, backward, gwq, gwk, s);
    return launch<__half>(a, backward, gwq, gwk, s);
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
    return launch_typed(a, false, nullptr, nullptr, stream);
}

int64_t cf_qk_norm_bwd_workspace_bytes(const cf_qk_norm *args)
{
    if (check_args("cf_qk_norm_bwd_workspace_bytes", args) != CF_OK) return 0;
    int single = 0;
    const int units = units_of(*args, true, single);
    // blocks of at least eight heads' lanes each; the most that a launch of any vector width has
    long long blocks = bwd_blocks(args->N * units, THREADS / 32);
    const long long least = (units + THREADS / 32 - 1) / (THREADS / 32);
    if (blocks < least) blocks = least;
    return (int64_t)((size_t)blocks * 2 * units * args->D * sizeof(float));
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
    return launch_typed(a, true, gwq, gwk, stream);
}

}  // extern "C"
