// The clipped policy loss and the preference loss on logits, forward and backward.
//
// Both need, for each row z of logits and its label a, the log probability lp = z_a - max - log(sum exp(z - max)),
// and both have the gradient dz_j = c (1[j = a] - exp(z_j - max) / sum) with one number c a row. So one kernel
// makes lp and the pair (max, 1 / sum) of every row in one read of the logits (a running maximum and sum), a
// little arithmetic on rows gives the loss and c, and one kernel reads the logits again and writes the gradient:
// 4 bytes a logit forward, 8 backward, about one exponential each, so HBM bounds them. Rows that the mask leaves
// out are not read; their gradient is zeros.
//
// Many loads in flight are what both need. Rows of up to kSmallRow logits belong to 1 to 32 lanes with several
// rows of a warp's run in flight (200000 rows of 61 logits, both passes: 51 us; a warp a row took 187); rows of some
// thousand logits to a warp, the long ones to a block of 256 threads (8 vectors in flight a thread forward, 16
// backward: 4096 rows of 50001 logits 151 and 252 us, 0.82 and 1.64 GB at the copy rate 125 and 250; forward 5 to 30%
// longer with 4 vectors, with a second set of vectors fetched while the first is summed, or with the logits brought to
// shared memory by bulk copies, as each leaves fewer warps to the arithmetic; 139 with the approximate exponential).
// A few very long rows are split among warps, and a second launch joins the parts. Statistics of up to 32 rows wait in
// a warp's lanes, so that the double precision arithmetic of the loss runs once for all of them and not once a row.
// Backward deals rows out as blocks end (uncounted rows cost a third, so dealing them out in advance leaves SMs idle:
// with a mask 418 instead of 352 us) and starts with the last long row, whose logits the forward pass may have left in
// L2. Log probabilities and everything behind them that can cancel (log ratios, the KL term, sums over tokens and rows)
// are held in 64 bits, a row's ratio and its product with the advantage in 32; sums run in a fixed order.
#include <math.h>

#include "k_common.cuh"

using namespace nck;

namespace {

constexpr int kSmallRow = 512, kShortRow = 1024; // rows read in one go by lanes, by a warp
constexpr float kNone = -INFINITY;

// e^x of the gradient by the approximate power of two: off by 2 steps and the rounding of x log2 e; results below
// 2^-126 are 0.
__device__ __forceinline__ float exp_of(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x * 1.4426950408889634f));
    return r;
}

// two floats at once (one issue slot for both)
__device__ __forceinline__ uint64_t two(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ uint64_t two(float x) { return two(x, x); }
__device__ __forceinline__ void apart(uint64_t v, float &x, float &y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

__device__ __forceinline__ float at_least(float x, float low) { // NaN stays NaN
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(x), "f"(low));
    return y;
}

// e^x of the sums, two x <= 0 at once: 2^n times a polynomial in f = x log2 e - n, |f| <= 1/2 (interpolation of
// (2^f - 1) / f at Chebyshev nodes). It is off by less than 1.5 * 2^-24 and, what matters here, by 7e-10 in the mean:
// with the approximate power a log probability is 5e-8 to 2e-7 too large in the mean (vocabularies of 96 to 128000),
// which adds up over the tokens of an answer. x below -87 counts as -87 (2e-38 of the largest term); NaN stays NaN.
__device__ __forceinline__ uint64_t exp_sum2(uint64_t x) {
    constexpr float kLog2e = 1.4426950408889634f, kRest = (float)(1.4426950408889634 - (double)kLog2e);
    constexpr float kRound = 12582912.0f + 127.0f; // adding it rounds to whole numbers; low bits: the number + 127
    float x0, x1, t0, t1;
    apart(x, x0, x1);
    const uint64_t y = two(at_least(x0, -87.0f), at_least(x1, -87.0f));
    const uint64_t t = fma2(y, two(kLog2e), two(kRound));
    const uint64_t f = fma2(y, two(kRest), fma2(y, two(kLog2e), fma2(t, two(-1.0f), two(kRound))));
    uint64_t p = fma2(f, two(0.00015453163f), two(0.0013390863f));
    p = fma2(p, f, two(0.009618083f));
    p = fma2(p, f, two(0.05550357f));
    p = fma2(p, f, two(0.2402265f));
    p = fma2(p, f, two(0.6931472f));
    apart(t, t0, t1);
    return mul2(fma2(p, f, two(1.0f)), two(__uint_as_float(__float_as_uint(t0) << 23), __uint_as_float(__float_as_uint(t1) << 23)));
}

__device__ __forceinline__ void exp_sum(float x, float y, float &ex, float &ey) { apart(exp_sum2(two(x, y)), ex, ey); }

struct Stat {
    float m, s; // running maximum, and the sum of exp(z - m)
};

// adds a maximum / sum pair to another; a side without finite values adds nothing
__device__ __forceinline__ Stat join(Stat a, Stat b) {
    const float m = fmaxf(a.m, b.m), base = m == kNone ? 0.0f : m;
    float ea, eb;
    exp_sum(a.m - base, b.m - base, ea, eb);
    return {m, fmaf(a.s, ea, b.s * eb)};
}

template <int N>
__device__ __forceinline__ void take(Stat &st, const float (&v)[N]) {
    static_assert(N % 2 == 0, "pairs");
    float top = v[0];
#pragma unroll
    for (int i = 1; i < N; i++) top = fmaxf(top, v[i]);
    const float m = fmaxf(st.m, top), base = m == kNone ? 0.0f : m;
    const uint64_t down = two(-base);
    uint64_t sum = exp_sum2(add2(two(v[0], v[1]), down));
#pragma unroll
    for (int i = 2; i < N; i += 2) sum = add2(sum, exp_sum2(add2(two(v[i], v[i + 1]), down)));
    if (m != st.m) { // (rarely, once a row's largest values have been met)
        float e, unused;
        exp_sum(st.m - base, 0.0f, e, unused);
        st.s *= e;
    }
    float x, y;
    apart(sum, x, y);
    st.m = m;
    st.s += x + y;
}

// floats before the first 16-byte boundary at or behind p, at most n
__device__ __forceinline__ int64_t lead_of(const float *p, int64_t n) {
    const int64_t k = (int64_t)((16 - ((uintptr_t)p & 15)) & 15) >> 2;
    return k < n ? k : n;
}

// Vectors before part k of n of a row's nv (V < 2^31, so nv < 2^29, and there are at most nv / 8 parts).
__device__ __forceinline__ int part_begin(int nv, int k, int n) { return n == 1 ? (k ? nv : 0) : (int)((int64_t)nv * k / n); }

// A team of W threads (t of them) reads part k of n of a row: U vectors in flight each.
template <int W, int U>
__device__ __forceinline__ Stat read_row(const float *z, int64_t V, int t, int k, int n) {
    Stat st = {kNone, 0.0f};
    const int64_t lead = lead_of(z, V);
    const int nv = (int)((V - lead) >> 2), end = part_begin(nv, k + 1, n);
    const float4 *z4 = reinterpret_cast<const float4 *>(z + lead);
    int i = part_begin(nv, k, n) + t;
    for (; i + (U - 1) * W < end; i += W * U) {
        float4 f[U];
        float v[4 * U];
#pragma unroll
        for (int u = 0; u < U; u++) f[u] = z4[i + u * W];
#pragma unroll
        for (int u = 0; u < U; u++) v[4 * u] = f[u].x, v[4 * u + 1] = f[u].y, v[4 * u + 2] = f[u].z, v[4 * u + 3] = f[u].w;
        take(st, v);
    }
    if (i < end) { // the rest, at most U - 1 vectors a thread
        float4 f[U - 1 > 0 ? U - 1 : 1];
#pragma unroll
        for (int u = 0; u < U - 1; u++) f[u] = i + u * W < end ? z4[i + u * W] : make_float4(kNone, kNone, kNone, kNone);
#pragma unroll
        for (int u = 0; u < U - 1; u++) {
            const float v[4] = {f[u].x, f[u].y, f[u].z, f[u].w};
            if (i + u * W < end) take(st, v);
        }
    }
    if (k) return st; // part 0 has the ends that are no whole vectors
    const int64_t tail = lead + 4 * (int64_t)nv;
    if (t < 3) {
        const float v[2] = {t < lead ? z[t] : kNone, t < V - tail ? z[tail + t] : kNone};
        take(st, v);
    }
    return st;
}

// A warp reads a row of up to kShortRow logits, all of it in flight at once.
__device__ __forceinline__ Stat read_short_row(const float *z, int V, int lane) {
    constexpr int U = kShortRow / 128;
    const int lead = (int)lead_of(z, V), nv = (V - lead) >> 2, tail = lead + 4 * nv;
    const float4 *z4 = reinterpret_cast<const float4 *>(z + lead);
    float4 f[U];
    const float v0[2] = {lane < lead ? z[lane] : kNone, lane < V - tail ? z[tail + lane] : kNone};
#pragma unroll
    for (int u = 0; u < U; u++)
        f[u] = lane + 32 * u < nv ? z4[lane + 32 * u] : make_float4(kNone, kNone, kNone, kNone);
    Stat st = {kNone, 0.0f};
    take(st, v0);
#pragma unroll
    for (int u = 0; u < U; u++) {
        if (32 * u >= nv) break;
        const float v[4] = {f[u].x, f[u].y, f[u].z, f[u].w};
        take(st, v);
    }
    return st;
}

// The statistics of W neighbouring lanes together, in all of them: the maximum first, so each sum is brought to it once.
template <int W = 32>
__device__ __forceinline__ Stat warp_join(Stat st) {
    float m = st.m;
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
    float e, unused;
    exp_sum(st.m - (m == kNone ? 0.0f : m), 0.0f, e, unused);
    float s = st.s * e;
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
    return {m, s};
}

// The statistics of the values that W neighbouring lanes hold, in all of them.
template <int W, int N>
__device__ __forceinline__ Stat lanes_stat(const float (&v)[N]) {
    static_assert(N % 2 == 0, "pairs");
    float m = v[0];
#pragma unroll
    for (int i = 1; i < N; i++) m = fmaxf(m, v[i]);
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
    const uint64_t down = two(m == kNone ? 0.0f : -m);
    uint64_t sum = exp_sum2(add2(two(v[0], v[1]), down));
#pragma unroll
    for (int i = 2; i < N; i += 2) sum = add2(sum, exp_sum2(add2(two(v[i], v[i + 1]), down)));
    float x, y;
    apart(sum, x, y);
    float s = x + y;
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
    return {m, s};
}

__device__ __forceinline__ const float *row_of(const nck_rows &q, int64_t r) {
    if (q.T == q.N) return q.z + r * q.st;
    const int64_t b = r / q.T;
    return q.z + b * q.sb + (r - b * q.T) * q.st;
}

__device__ __forceinline__ bool counted(const nck_rows &q, int64_t r) { return !q.mask || q.mask[r] != 0; }

struct Sums {
    double loss, count;
};

// What a row has besides its statistics: the label's logit and the loss's inputs. The row is read as label 0 (and
// reported) when its label is out of range.
struct RowIn {
    float z, old, ref, adv;
};

__device__ __forceinline__ RowIn row_in(const nck_rows &q, const nck_policy &p, int64_t r) {
    int32_t a = q.lab[r];
    if (a < 0 || a >= q.V) {
        report(q.status, NCK_ERR_LABEL);
        a = 0;
    }
    RowIn in = {row_of(q, r)[a], 0.0f, 0.0f, 0.0f};
    if (p.adv) {
        in.old = p.old[r], in.adv = p.adv[r];
        if (p.kl != 0.0f) in.ref = p.ref[r];
    }
    return in;
}

// e^a - 1 - a from e = e^a - 1, never negative: the two cancel near 0 (a policy near its reference), where the series'
// next term is below 2^-29 of the sum, and both are infinite for an action of probability 0.
__device__ __forceinline__ double exp_rest(double a, double e) {
    if (fabs(a) < 1.220703125e-4) return a * a * (0.5 + a * (1.0 / 6.0)); // 2^-13
    return isinf(e) ? e : e - a;
}

// What a row's log probability becomes: its loss term and the factor c of its gradient (without 1 / count).
__device__ __forceinline__ double policy_term(const nck_policy &p, const RowIn &in, double lp, float *c) {
    const float A = in.adv, ratio = expf((float)(lp - (double)in.old));
    const float lo = 1.0f - p.clip_low, hi = 1.0f + p.clip_high;
    const float held = fminf(fmaxf(ratio, lo), hi);
    const float gain = fminf(ratio * A, held * A);
    const bool moves = A >= 0.0f ? ratio <= hi : ratio >= lo, lost = isnan(ratio) || isnan(A);
    double term = lost ? ratio + A : -gain;
    float f = lost ? ratio + A : moves ? -A * ratio : 0.0f;
    if (p.kl != 0.0f) {
        const double away = (double)in.ref - lp, e = expm1(away);
        term += (double)p.kl * exp_rest(away, e);
        f -= p.kl * (float)e;
    }
    *c = f;
    return term;
}

__device__ __forceinline__ Sums finish_row(const nck_rows &q, const nck_policy &p, int64_t r, Stat st, const RowIn &in) {
    const double lp = ((double)in.z - (double)st.m) - log((double)st.s);
    if (q.stat) reinterpret_cast<float2 *>(q.stat)[r] = make_float2(st.m, 1.0f / st.s);
    if (q.lp64) q.lp64[r] = lp;
    if (q.lp32) q.lp32[r] = (float)lp;
    if (!p.adv) return {0.0, 1.0};
    float c;
    const double term = policy_term(p, in, lp, &c);
    if (p.coef) p.coef[r] = c;
    return {term, 1.0};
}

__device__ __forceinline__ void skip_row(const nck_rows &q, const nck_policy &p, int64_t r) {
    if (q.lp64) q.lp64[r] = 0.0;
    if (q.lp32) q.lp32[r] = 0.0f;
    if (p.coef) p.coef[r] = 0.0f;
}

// The sums of a block's threads, in thread 0.
__device__ Sums block_sums(Sums mine) {
    __shared__ double2 red[8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        mine.loss += __shfl_xor_sync(~0u, mine.loss, o);
        mine.count += __shfl_xor_sync(~0u, mine.count, o);
    }
    __syncthreads();
    if (lane == 0) red[warp] = make_double2(mine.loss, mine.count);
    __syncthreads();
    mine = {0.0, 0.0};
    if (threadIdx.x == 0)
        for (int w = 0; w < warps; w++) mine.loss += red[w].x, mine.count += red[w].y;
    return mine;
}

// Loss and 1 / count, from thread 0's sums.
__device__ void write_loss(const nck_policy &p, Sums all) {
    if (threadIdx.x) return;
    const double n = all.count > 1.0 ? all.count : 1.0;
    *p.loss = (float)(all.loss / n);
    if (p.scale) *p.scale = (float)(1.0 / n);
}

// The same from every block's sums, in block order, by the block that ends last.
__device__ void finish_loss(const nck_policy &p, Sums mine, double2 *part, unsigned *counter) {
    mine = block_sums(mine);
    if (threadIdx.x == 0) part[blockIdx.x] = make_double2(mine.loss, mine.count);
    if (!last_block_done(counter)) return;
    mine = {0.0, 0.0};
    for (int b = threadIdx.x; b < (int)gridDim.x; b += blockDim.x) {
        const double2 v = __ldcg(part + b);
        mine.loss += v.x, mine.count += v.y;
    }
    write_loss(p, block_sums(mine));
}

// One warp a run of `run` rows, row i's statistics in lane i.
__global__ void __launch_bounds__(256) k_rows_warp(nck_rows q, nck_policy p, int run, double2 *part, unsigned *counter) {
    cudaGridDependencySynchronize();
    const int lane = threadIdx.x & 31;
    const int64_t warps = (int64_t)gridDim.x * 8;
    Sums sums = {0.0, 0.0};
    for (int64_t r0 = ((int64_t)blockIdx.x * 8 + (threadIdx.x >> 5)) * run; r0 < q.N; r0 += warps * run) {
        const int n = q.N - r0 < run ? (int)(q.N - r0) : run;
        const bool live = lane < n && counted(q, r0 + lane);
        const unsigned any = __ballot_sync(~0u, live);
        Stat own = {kNone, 0.0f};
        RowIn in = {};
        if (live) in = row_in(q, p, r0 + lane); // on its way while the rows are read
        for (int k = 0; k < n; k++) {
            if (!(any >> k & 1)) continue;
            const float *z = row_of(q, r0 + k);
            const Stat st = warp_join(q.V <= kShortRow ? read_short_row(z, (int)q.V, lane) : read_row<32, 8>(z, q.V, lane, 0, 1));
            if (lane == k) own = st;
        }
        if (live) {
            const Sums s = finish_row(q, p, r0 + lane, own, in);
            sums.loss += s.loss, sums.count += s.count;
        } else if (lane < n) {
            skip_row(q, p, r0 + lane);
        }
    }
    if (p.loss) finish_loss(p, sums, part, counter);
}

// Rows of up to E G logits: G lanes a row, 32 / G rows a pass and P passes of a warp's run in flight; row i's
// statistics go to lane i.
template <int G, int E, int P>
__global__ void __launch_bounds__(256) k_rows_small(nck_rows q, nck_policy p, int run, double2 *part, unsigned *counter) {
    cudaGridDependencySynchronize();
    constexpr int R = 32 / G;
    const int lane = threadIdx.x & 31, l = lane % G, V = (int)q.V;
    const int64_t warps = (int64_t)gridDim.x * 8;
    Sums sums = {0.0, 0.0};
    for (int64_t r0 = ((int64_t)blockIdx.x * 8 + (threadIdx.x >> 5)) * run; r0 < q.N; r0 += warps * run) {
        const int n = q.N - r0 < run ? (int)(q.N - r0) : run;
        const bool live = lane < n && counted(q, r0 + lane);
        const unsigned any = __ballot_sync(~0u, live);
        Stat own = {kNone, 0.0f};
        RowIn in = {};
        if (live) in = row_in(q, p, r0 + lane);
        for (int it = 0; it * R < n; it += P) {
            float v[P][E];
#pragma unroll
            for (int u = 0; u < P; u++) {
                const int row = (it + u) * R + lane / G;
                const bool ok = row < n && (any >> row & 1);
                const float *z = row_of(q, r0 + (ok ? row : 0));
#pragma unroll
                for (int e = 0; e < E; e++) v[u][e] = ok && e * G + l < V ? z[e * G + l] : kNone;
            }
#pragma unroll
            for (int u = 0; u < P; u++) {
                const Stat st = lanes_stat<G>(v[u]);
                const int from = lane % R * G;
                const Stat mine = {__shfl_sync(~0u, st.m, from), __shfl_sync(~0u, st.s, from)};
                if (lane / R == it + u) own = mine;
            }
        }
        if (live) {
            const Sums s = finish_row(q, p, r0 + lane, own, in);
            sums.loss += s.loss, sums.count += s.count;
        } else if (lane < n) {
            skip_row(q, p, r0 + lane);
        }
    }
    if (p.loss) finish_loss(p, sums, part, counter);
}

// A block a row. Statistics of counted rows wait in the lanes of the first warp, which finishes 32 at a time.
__global__ void __launch_bounds__(256) k_rows_block(nck_rows q, nck_policy p, double2 *part, unsigned *counter) {
    cudaGridDependencySynchronize();
    __shared__ Stat red[2][8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Sums sums = {0.0, 0.0};
    Stat own = {kNone, 0.0f};
    RowIn in = {};
    int64_t own_row = -1;
    int turn = 0, held = 0;
    const auto finish = [&]() {
        if (own_row >= 0) {
            const Sums s = finish_row(q, p, own_row, own, in);
            sums.loss += s.loss, sums.count += s.count;
        }
        own_row = -1, held = 0;
    };
    for (int64_t r = blockIdx.x; r < q.N; r += gridDim.x) {
        if (!counted(q, r)) {
            if (threadIdx.x == 0) skip_row(q, p, r);
            continue;
        }
        const Stat st = warp_join(read_row<256, 8>(row_of(q, r), q.V, threadIdx.x, 0, 1));
        if (lane == 0) red[turn][warp] = st;
        __syncthreads();
        if (warp == 0) {
            Stat all = {kNone, 0.0f};
            if (lane < 8) all = red[turn][lane];
            all = warp_join(all);
            if (lane == held) own = all, own_row = r, in = row_in(q, p, r);
            if (++held == 32) finish();
        }
        turn ^= 1;
    }
    if (warp == 0) finish();
    if (p.loss) finish_loss(p, sums, part, counter);
}

// Few rows: a warp takes parts of rows, with no barrier between warps; k_rows_finish joins them.
__global__ void __launch_bounds__(256) k_rows_parts(nck_rows q, int parts, float2 *part) {
    cudaGridDependencySynchronize();
    const int lane = threadIdx.x & 31;
    for (int64_t it = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); it < q.N * parts; it += (int64_t)gridDim.x * 8) {
        const int64_t r = it / parts;
        if (!counted(q, r)) continue;
        const Stat all = warp_join(read_row<32, 8>(row_of(q, r), q.V, lane, (int)(it - r * parts), parts));
        if (lane == 0) part[it] = make_float2(all.m, all.s);
    }
}

// A warp a run of rows: their parts joined, row i's in lane i, and the rows finished.
__global__ void __launch_bounds__(256) k_rows_finish(nck_rows q, nck_policy p, int parts, int run, const float2 *part,
                                                     double2 *sums_of, unsigned *counter) {
    cudaGridDependencySynchronize();
    const int lane = threadIdx.x & 31;
    Sums sums = {0.0, 0.0};
    const int64_t r0 = ((int64_t)blockIdx.x * 8 + (threadIdx.x >> 5)) * run;
    const int n = q.N - r0 < run ? (int)(q.N - r0) : run;
    const bool live = lane < n && counted(q, r0 + lane);
    const unsigned any = __ballot_sync(~0u, live);
    Stat own = {kNone, 0.0f};
    RowIn in = {};
    if (live) in = row_in(q, p, r0 + lane);
    for (int i = 0; i < n; i++) {
        if (!(any >> i & 1)) continue;
        Stat st = {kNone, 0.0f};
        for (int k = lane; k < parts; k += 32) {
            const float2 v = __ldcg(part + (r0 + i) * parts + k);
            st = join(st, {v.x, v.y});
        }
        st = warp_join(st);
        if (lane == i) own = st;
    }
    if (live) {
        const Sums s = finish_row(q, p, r0 + lane, own, in);
        sums.loss += s.loss, sums.count += s.count;
    } else if (lane < n) {
        skip_row(q, p, r0 + lane);
    }
    if (p.loss) finish_loss(p, sums, sums_of, counter);
}

// Sums of a pair's two sequences, the pair's loss term and its sequences' factors; the last block sums the terms.
__global__ void __launch_bounds__(256) k_pairs(nck_pairs p, const double *lp, double *term, unsigned *counter) {
    cudaGridDependencySynchronize();
    __shared__ double red[2][8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t i = blockIdx.x;
    for (int k = 0; k < 2; k++) {
        const double *x = lp + (i + k * p.P) * p.T;
        double s = 0.0;
        for (int64_t t = threadIdx.x; t < p.T; t += blockDim.x) s += x[t];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
        if (lane == 0) red[k][warp] = s;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        double seq[2] = {0.0, 0.0};
        for (int k = 0; k < 2; k++) {
            for (int w = 0; w < 8; w++) seq[k] += red[k][w];
            if (p.seq) p.seq[i + k * p.P] = (float)seq[k];
            if (p.ref) seq[k] -= (double)p.ref[i + k * p.P];
        }
        const double h = (double)p.beta * (seq[0] - seq[1]), eps = (double)p.smoothing;
        const double soft = log1p(exp(-fabs(h)));  // softplus(-|h|)
        double loss = (1.0 - eps) * (soft + (h < 0.0 ? -h : 0.0));
        if (eps > 0.0) loss += eps * (soft + (h > 0.0 ? h : 0.0)); // (an infinite h times a weight of 0 is NaN)
        term[i] = loss;
        if (p.coef) {
            const double c = (double)p.beta / (double)p.P * (1.0 / (1.0 + exp(-h)) - (1.0 - eps));
            p.coef[i] = (float)c;
            p.coef[i + p.P] = (float)-c;
        }
    }
    if (!last_block_done(counter)) return;
    double s = 0.0;
    for (int64_t j = threadIdx.x; j < p.P; j += blockDim.x) s += __ldcg(term + j);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
    if (lane == 0) red[0][warp] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        s = 0.0;
        for (int w = 0; w < 8; w++) s += red[0][w];
        *p.loss = (float)(s / (double)p.P);
    }
}

// The gradient of part k of n of a row by a team of W threads: dst (+)= c (1[j = a] - exp(z - m) inv).
template <int W, int U, bool ACC>
__device__ __forceinline__ void grad_row(const float *z, float *dst, int64_t V, float c, float m, float inv, int64_t a, int t,
                                         int k, int n) {
    const bool even = (((uintptr_t)z ^ (uintptr_t)dst) & 15) == 0; // the row and its gradient share their boundaries
    const bool blank = c == 0.0f;                                  // nothing of the row is read
    if (ACC && blank) return;
    const int64_t lead = lead_of(dst, V);
    const int nv = (int)((V - lead) >> 2), end = part_begin(nv, k + 1, n);
    const int64_t tail = lead + 4 * (int64_t)nv;
    float4 *d4 = reinterpret_cast<float4 *>(dst + lead);
    const float f = -c * inv;
    const auto one = [&](int64_t j) {
        float v = blank ? 0.0f : f * exp_of(z[j] - m);
        if (j == a) v += c;
        dst[j] = ACC ? dst[j] + v : v;
    };
    if (k == 0) {
        if (t < lead) one(t);
        if (t < V - tail) one(tail + t);
    }
    int i = part_begin(nv, k, n) + t;
    if (blank) {
        for (; i < end; i += W) d4[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        return;
    }
    const float *from = z + lead;
    const int64_t hot = a - lead; // the label's place among the vectors' floats
    const auto fetch = [&](int j) {
        const float *at = from + 4 * (int64_t)j;
        return even ? *reinterpret_cast<const float4 *>(at) : make_float4(at[0], at[1], at[2], at[3]);
    };
    const auto give = [&](int j, float4 v, float4 old) {
        float4 g = make_float4(f * exp_of(v.x - m), f * exp_of(v.y - m), f * exp_of(v.z - m), f * exp_of(v.w - m));
        const uint64_t w = (uint64_t)(hot - 4 * (int64_t)j);
        if (w < 4) g.x += w == 0 ? c : 0.0f, g.y += w == 1 ? c : 0.0f, g.z += w == 2 ? c : 0.0f, g.w += w == 3 ? c : 0.0f;
        if (ACC) g.x += old.x, g.y += old.y, g.z += old.z, g.w += old.w;
        d4[j] = g;
    };
    for (; i < end; i += W * U) {
        float4 v[U], old[ACC ? U : 1] = {};
#pragma unroll
        for (int u = 0; u < U; u++)
            if (i + u * W < end) {
                v[u] = fetch(i + u * W);
                if (ACC) old[ACC ? u : 0] = d4[i + u * W];
            }
#pragma unroll
        for (int u = 0; u < U; u++)
            if (i + u * W < end) give(i + u * W, v[u], old[ACC ? u : 0]);
    }
}

template <int W, bool ACC>
__global__ void __launch_bounds__(256) k_rows_grad(nck_rows q, nck_rows_grad g, int parts) {
    cudaGridDependencySynchronize();
    const int t = threadIdx.x % W;
    const float up = g.up[0] * (g.scale ? g.scale[0] : 1.0f);
    const int64_t teams = (int64_t)gridDim.x * (256 / W);
    // from the last row back: what the forward pass read last is still in L2
    for (int64_t it = (int64_t)blockIdx.x * (256 / W) + threadIdx.x / W; it < q.N * parts; it += teams) {
        const int64_t turn = parts == 1 ? it : it / parts, r = q.N - 1 - turn;
        const float c = counted(q, r) ? up * g.coef[r / g.per_coef] : 0.0f;
        const float2 st = c == 0.0f ? make_float2(0.f, 0.f) : reinterpret_cast<const float2 *>(q.stat)[r];
        int64_t a = q.lab[r];
        if (a < 0 || a >= q.V) a = 0;
        grad_row<W, W == 32 || ACC ? 8 : 16, ACC>(row_of(q, r), g.dz + r * q.V, q.V, c, st.x, st.y, a, t, (int)(it - turn * parts), parts);
    }
}

// The gradient of rows of up to E G logits, G lanes a row: a warp takes a run of rows, lane i fetching what row i needs.
template <int G, int E, int P, bool ACC>
__global__ void __launch_bounds__(256) k_rows_grad_small(nck_rows q, nck_rows_grad g, int run) {
    constexpr int R = 32 / G;
    cudaGridDependencySynchronize();
    const int lane = threadIdx.x & 31, l = lane % G, V = (int)q.V;
    const float up = g.up[0] * (g.scale ? g.scale[0] : 1.0f);
    const int64_t r0 = ((int64_t)blockIdx.x * 8 + (threadIdx.x >> 5)) * run;
    if (r0 >= q.N) return;
    const int n = q.N - r0 < run ? (int)(q.N - r0) : run;
    float c = 0.0f;
    float2 st = make_float2(0.0f, 0.0f);
    int a = 0;
    if (lane < n) {
        const int64_t r = r0 + lane;
        if (counted(q, r)) c = up * g.coef[r / g.per_coef];
        if (c != 0.0f) {
            st = reinterpret_cast<const float2 *>(q.stat)[r];
            a = q.lab[r];
            if (a < 0 || a >= V) a = 0;
        }
    }
    for (int it = 0; it * R < n; it += P) {
        float v[P][E], old[ACC ? P : 1][ACC ? E : 1];
#pragma unroll
        for (int u = 0; u < P; u++) {
            const int row = (it + u) * R + lane / G;
            const float rc = __shfl_sync(~0u, c, row & 31);
            const bool ok = row < n, read = ok && rc != 0.0f;
            const float *z = row_of(q, r0 + (ok ? row : 0));
            const float *dz = g.dz + (r0 + (ok ? row : 0)) * V;
#pragma unroll
            for (int e = 0; e < E; e++) {
                v[u][e] = read && e * G + l < V ? z[e * G + l] : kNone;
                if (ACC) old[ACC ? u : 0][ACC ? e : 0] = read && e * G + l < V ? dz[e * G + l] : 0.0f;
            }
        }
#pragma unroll
        for (int u = 0; u < P; u++) {
            const int row = (it + u) * R + lane / G, s = row & 31;
            const float rc = __shfl_sync(~0u, c, s), m = __shfl_sync(~0u, st.x, s), inv = __shfl_sync(~0u, st.y, s);
            const int ra = __shfl_sync(~0u, a, s);
            if (row >= n || (ACC && rc == 0.0f)) continue;
            float *dz = g.dz + (r0 + row) * V;
#pragma unroll
            for (int e = 0; e < E; e++) {
                const int j = e * G + l;
                if (j >= V) break;
                float d = rc == 0.0f ? 0.0f : -rc * inv * exp_of(v[u][e] - m);
                if (j == ra) d += rc;
                dz[j] = ACC ? old[ACC ? u : 0][ACC ? e : 0] + d : d;
            }
        }
    }
}

// Parts of a row of V logits so that `rows` rows make about `items` parts, none below `least` logits.
int parts_for(int64_t rows, int64_t V, int64_t items, int64_t least) {
    int64_t n = (items + rows - 1) / rows;
    if (n > V / least) n = V / least;
    return n < 1 ? 1 : (int)n;
}

// Blocks of a grid-stride launch: one full wave of the kernel, or fewer for less work.
template <typename K>
int wave_of(const nck_dev *d, K kernel, int *room) {
    if (!*room) *room = resident_blocks(d, kernel, 256);
    return *room;
}

int at_most(int64_t want, int room) { return (int)(want < 1 ? 1 : want < room ? want : room); }

template <int W, bool ACC>
void launch_grad(nck_dev *d, const nck_rows *q, const nck_rows_grad *g) {
    static int room = 0;
    wave_of(d, k_rows_grad<W, ACC>, &room);
    const int parts = W == 32 ? 1 : parts_for(q->N, q->V, room, 4096);
    launch_early(d, k_rows_grad<W, ACC>, at_most((q->N * parts + 256 / W - 1) / (256 / W), 1 << 30), 256, *q, *g, parts);
    NCK_LAUNCHED(d, 1);
}

// Whether a row belongs to a warp and not to a block: short rows, and middling ones when there are enough of them
// to fill the GPU with warps. Both passes, warp and block: 50000 rows of 1500 logits 177 and 745 us, 500 rows 14.6
// and 17.6; 2000 rows of 8000 46 and 56 us, 500 rows 31 and 23; 8192 rows of 16000 281 and 273.
bool warp_rows(const nck_rows *q) { return q->V <= 2048 || (q->V <= 12288 && q->N >= 1024); }

// Rows to a warp: as few as fill the resident warps, at most 32.
int run_for(const nck_dev *d, int64_t rows, int room) {
    const int64_t run = (rows + (int64_t)room * 8 - 1) / ((int64_t)room * 8);
    return (int)(run < 1 ? 1 : run > 32 ? 32 : run);
}

template <int G, int E, int P>
void launch_small(nck_dev *d, const nck_rows *q, const nck_policy *p, const nck_rows_grad *g) {
    static int room = 0;
    wave_of(d, k_rows_small<G, E, P>, &room);
    constexpr int R = 32 / G;
    const int run = (run_for(d, q->N, room) + R - 1) / R * R; // whole passes
    const int64_t blocks = (q->N + run * 8 - 1) / (run * 8);
    if (p) launch_early(d, k_rows_small<G, E, P>, at_most(blocks, room), 256, *q, *p, run, (double2 *)d->scratch, d->counters);
    else if (g->acc) launch_early(d, k_rows_grad_small<G, E, P, true>, blocks, 256, *q, *g, run);
    else launch_early(d, k_rows_grad_small<G, E, P, false>, blocks, 256, *q, *g, run);
    NCK_LAUNCHED(d, 1);
}

// Rows of up to kSmallRow logits, forward (p) or backward (g).
void dispatch_small(nck_dev *d, const nck_rows *q, const nck_policy *p, const nck_rows_grad *g) {
    if (q->V <= 4) launch_small<1, 4, 4>(d, q, p, g);
    else if (q->V <= 8) launch_small<2, 4, 4>(d, q, p, g);
    else if (q->V <= 16) launch_small<4, 4, 4>(d, q, p, g);
    else if (q->V <= 32) launch_small<8, 4, 4>(d, q, p, g);
    else if (q->V <= 64) launch_small<16, 4, 4>(d, q, p, g);
    else if (q->V <= 128) launch_small<32, 4, 4>(d, q, p, g);
    else if (q->V <= 256) launch_small<32, 8, 3>(d, q, p, g);
    else launch_small<32, 16, 1>(d, q, p, g);
}

}  // namespace

extern "C" void nck_rows_logp(nck_dev *d, const nck_rows *q, const nck_policy *p) {
    static int room_warp = 0, room_block = 0, room_parts = 0;
    nck_rows rows = *q;
    rows.status = d->status;
    nck_policy pol;
    if (p) pol = *p;
    else pol = nck_policy{};
    Scope sc(d, "logits_logp", 4.0 * q->N * q->V, 4.0 * q->N * q->V);
    double2 *part = (double2 *)d->scratch;
    if (q->V <= kSmallRow) {
        dispatch_small(d, &rows, &pol, nullptr);
        return;
    }
    NCK_LAUNCHED(d, 1);
    if (warp_rows(q)) {
        const int64_t run = run_for(d, q->N, wave_of(d, k_rows_warp, &room_warp));
        launch_early(d, k_rows_warp, at_most((q->N + run * 8 - 1) / (run * 8), room_warp), 256, rows, pol, (int)run, part, d->counters);
        return;
    }
    wave_of(d, k_rows_block, &room_block);
    // Parts of rows when an SM would have only a few rows and they are long, as the blocks that get one more row hold up
    // the rest (parts and blocks, us: of 128000 logits 61 rows 15 and 30, 244 35 and 42, 488 52 and 59, 1464 125 and
    // 130, 1952 169 and 166; of 256000 488 rows 89 and 108; of 65536 488 rows 35 and 35, 976 53 and 51; of 50001 61 rows
    // 12.5 and 14).
    if (q->V < 65536 || q->N >= d->sm_count * (q->V < 80000 ? (int64_t)2 : 10) || q->N == 0) {
        launch_early(d, k_rows_block, at_most(q->N, room_block), 256, rows, pol, part, d->counters);
        return;
    }
    wave_of(d, k_rows_parts, &room_parts);
    const int parts = parts_for(q->N, q->V, (int64_t)room_parts * 8 * 2, 4096);
    float2 *stats = (float2 *)(part + 4096); // behind the finishing blocks' sums
    launch_early(d, k_rows_parts, at_most((q->N * parts + 7) / 8, room_parts), 256, rows, parts, stats);
    const int64_t run = (q->N + 4096 * 8 - 1) / (4096 * 8); // (few rows: one)
    launch_early(d, k_rows_finish, (q->N + run * 8 - 1) / (run * 8), 256, rows, pol, parts, (int)run, (const float2 *)stats, part,
                 d->counters);
    NCK_LAUNCHED(d, 1);
}

extern "C" void nck_pref_pairs(nck_dev *d, const nck_pairs *p, const double *lp) {
    Scope sc(d, "preference_pairs", 0.0, 16.0 * p->P * p->T);
    launch_early(d, k_pairs, p->P, 256, *p, lp, p->term, d->counters);
    NCK_LAUNCHED(d, 1);
}

extern "C" void nck_rows_bwd(nck_dev *d, const nck_rows *q, const nck_rows_grad *g) {
    if (q->N == 0) return;
    Scope sc(d, "logits_logp_bwd", 4.0 * q->N * q->V, 8.0 * q->N * q->V);
    if (q->V <= kSmallRow) {
        dispatch_small(d, q, nullptr, g);
    } else if (warp_rows(q)) {
        if (g->acc) launch_grad<32, true>(d, q, g);
        else launch_grad<32, false>(d, q, g);
    } else {
        if (g->acc) launch_grad<256, true>(d, q, g);
        else launch_grad<256, false>(d, q, g);
    }
}
