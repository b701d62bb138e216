// The clipped policy loss and the preference loss on logits, forward and backward.
//
// Both need, for each row z of logits and its label a, the log probability lp = z_a - max - log(sum exp(z - max)),
// and both have the gradient dz_j = c (1[j = a] - exp(z_j - max) / sum) with one number c a row. So one kernel
// makes lp and the pair (max, 1 / sum) of every row in one read of the logits (a running maximum and sum), a
// little arithmetic on rows gives the loss and c, and one kernel reads the logits again and writes the gradient:
// 4 bytes a logit forward, 8 backward, about one exponential each, so HBM bounds them. Rows that the mask leaves
// out are not read; their gradient is zeros.
//
// A row of up to kWarpRow logits belongs to a warp, a longer one to a block of 256 threads. A warp takes a
// run of up to 32 rows and keeps the statistics of row i in lane i, so that the double precision arithmetic of
// the loss runs once a run and not once a row. Log probabilities and everything behind them that can cancel
// (log ratios, sums over tokens and rows) are held in 64 bits; sums run in a fixed order.
#include <math.h>

#include "k_common.cuh"

using namespace nck;

namespace {

constexpr int kWarpRow = 1024;
constexpr float kNone = -INFINITY;

struct Stat {
    float m, s; // running maximum, and the sum of exp(z - m)
};

// adds a maximum / sum pair to another; a side without finite values has s = 0
__device__ __forceinline__ Stat join(Stat a, Stat b) {
    const float m = fmaxf(a.m, b.m), base = m == kNone ? 0.0f : m;
    return {m, a.s * __expf(a.m - base) + b.s * __expf(b.m - base)};
}

template <int N>
__device__ __forceinline__ void take(Stat &st, const float (&v)[N]) {
    float top = v[0];
#pragma unroll
    for (int i = 1; i < N; i++) top = fmaxf(top, v[i]);
    const float m = fmaxf(st.m, top), base = m == kNone ? 0.0f : m;
    float s = st.s * __expf(st.m - base);
#pragma unroll
    for (int i = 0; i < N; i++) s += __expf(v[i] - base);
    st.m = m, st.s = s;
}

// floats before the first 16-byte boundary at or behind p, at most n
__device__ __forceinline__ int64_t lead_of(const float *p, int64_t n) {
    const int64_t k = (int64_t)((16 - ((uintptr_t)p & 15)) & 15) >> 2;
    return k < n ? k : n;
}

// A team of W threads (t of them) reads a row: U vectors in flight each.
template <int W, int U>
__device__ __forceinline__ Stat read_row(const float *z, int64_t V, int t) {
    Stat st = {kNone, 0.0f};
    const int64_t lead = lead_of(z, V), nv = (V - lead) >> 2;
    const float4 *z4 = reinterpret_cast<const float4 *>(z + lead);
    for (int64_t i = t; i < nv; i += W * U) {
        float v[4 * U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            float4 f = make_float4(kNone, kNone, kNone, kNone);
            if (i + u * W < nv) f = __ldg(z4 + i + u * W);
            v[4 * u] = f.x, v[4 * u + 1] = f.y, v[4 * u + 2] = f.z, v[4 * u + 3] = f.w;
        }
        take(st, v);
    }
    const int64_t tail = lead + 4 * nv;
    if (t < lead) {
        const float v[1] = {z[t]};
        take(st, v);
    }
    if (t < V - tail) {
        const float v[1] = {z[tail + t]};
        take(st, v);
    }
    return st;
}

__device__ __forceinline__ Stat warp_join(Stat st) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const Stat b = {__shfl_xor_sync(~0u, st.m, o), __shfl_xor_sync(~0u, st.s, o)};
        st = join(st, b);
    }
    return st;
}

// lp of a row in 64 bits; the row is read as label 0 (and reported) when its label is out of range
__device__ __forceinline__ double logp_of(const nck_rows &q, const float *z, int64_t r, Stat st) {
    int32_t a = q.lab[r];
    if (a < 0 || a >= q.V) {
        report(q.status, NCK_ERR_LABEL);
        a = 0;
    }
    return ((double)z[a] - (double)st.m) - log((double)st.s);
}

__device__ __forceinline__ const float *row_of(const nck_rows &q, int64_t r) {
    const int64_t b = r / q.T;
    return q.z + b * q.sb + (r - b * q.T) * q.st;
}

__device__ __forceinline__ bool counted(const nck_rows &q, int64_t r) { return !q.mask || q.mask[r] != 0; }

struct Sums {
    double loss, count;
};

// What a row's log probability becomes: its loss term and the factor c of its gradient (without 1 / count).
__device__ __forceinline__ double policy_term(const nck_policy &p, int64_t r, double lp, float *c) {
    const float A = p.adv[r], ratio = expf((float)(lp - (double)p.old[r]));
    const float lo = 1.0f - p.clip_low, hi = 1.0f + p.clip_high;
    const float held = fminf(fmaxf(ratio, lo), hi);
    const float gain = fminf(ratio * A, held * A);
    const bool moves = A >= 0.0f ? ratio <= hi : ratio >= lo;
    float term = isnan(ratio) ? ratio : -gain, f = moves ? -A * ratio : 0.0f;
    if (p.kl != 0.0f) {
        const float away = (float)((double)p.ref[r] - lp), e = expm1f(away);
        term += p.kl * (e - away);
        f -= p.kl * e;
    }
    *c = f;
    return (double)term;
}

__device__ __forceinline__ Sums finish_row(const nck_rows &q, const nck_policy &p, int64_t r, Stat st) {
    const double lp = logp_of(q, row_of(q, r), r, st);
    if (q.stat) reinterpret_cast<float2 *>(q.stat)[r] = make_float2(st.m, 1.0f / st.s);
    if (q.lp64) q.lp64[r] = lp;
    if (q.lp32) q.lp32[r] = (float)lp;
    if (!p.adv) return {0.0, 1.0};
    float c;
    const double term = policy_term(p, r, lp, &c);
    if (p.coef) p.coef[r] = c;
    return {term, 1.0};
}

__device__ __forceinline__ void skip_row(const nck_rows &q, const nck_policy &p, int64_t r) {
    if (q.lp64) q.lp64[r] = 0.0;
    if (q.lp32) q.lp32[r] = 0.0f;
    if (p.coef) p.coef[r] = 0.0f;
}

// Loss and 1 / count from every block's sums, in block order, by the block that ends last.
__device__ void finish_loss(const nck_policy &p, Sums mine, double2 *part, unsigned *counter) {
    __shared__ double2 red[8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int round = 0; round < 2; round++) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            mine.loss += __shfl_xor_sync(~0u, mine.loss, o);
            mine.count += __shfl_xor_sync(~0u, mine.count, o);
        }
        __syncthreads();
        if (lane == 0) red[warp] = make_double2(mine.loss, mine.count);
        __syncthreads();
        Sums all = {0.0, 0.0};
        for (int w = 0; w < 8; w++) all.loss += red[w].x, all.count += red[w].y;
        if (round) {
            if (threadIdx.x == 0) {
                const double n = all.count > 1.0 ? all.count : 1.0;
                *p.loss = (float)(all.loss / n);
                if (p.scale) *p.scale = (float)(1.0 / n);
            }
            return;
        }
        if (threadIdx.x == 0) part[blockIdx.x] = make_double2(all.loss, all.count);
        if (!last_block_done(counter)) return;
        mine = {0.0, 0.0};
        for (int b = threadIdx.x; b < (int)gridDim.x; b += blockDim.x) {
            const double2 v = __ldcg(part + b);
            mine.loss += v.x, mine.count += v.y;
        }
    }
}

// One warp a run of `run` rows, row i's statistics in lane i.
__global__ void __launch_bounds__(256) k_rows_warp(nck_rows q, nck_policy p, int run, double2 *part, unsigned *counter) {
    const int lane = threadIdx.x & 31;
    const int64_t warps = (int64_t)gridDim.x * 8;
    Sums sums = {0.0, 0.0};
    for (int64_t r0 = ((int64_t)blockIdx.x * 8 + (threadIdx.x >> 5)) * run; r0 < q.N; r0 += warps * run) {
        const int n = q.N - r0 < run ? (int)(q.N - r0) : run;
        const bool live = lane < n && counted(q, r0 + lane);
        const unsigned any = __ballot_sync(~0u, live);
        Stat own = {kNone, 0.0f};
        for (int i = 0; i < n; i++) {
            if (!(any >> i & 1)) continue;
            const Stat st = warp_join(read_row<32, 1>(row_of(q, r0 + i), q.V, lane));
            if (lane == i) own = st;
        }
        if (live) {
            const Sums s = finish_row(q, p, r0 + lane, own);
            sums.loss += s.loss, sums.count += s.count;
        } else if (lane < n) {
            skip_row(q, p, r0 + lane);
        }
    }
    if (p.loss) finish_loss(p, sums, part, counter);
}

// One block a row.
__global__ void __launch_bounds__(256) k_rows_block(nck_rows q, nck_policy p, double2 *part, unsigned *counter) {
    __shared__ Stat red[2][8];
    Sums sums = {0.0, 0.0};
    int turn = 0;
    for (int64_t r = blockIdx.x; r < q.N; r += gridDim.x) {
        if (!counted(q, r)) {
            if (threadIdx.x == 0) skip_row(q, p, r);
            continue;
        }
        const Stat st = warp_join(read_row<256, 4>(row_of(q, r), q.V, threadIdx.x));
        if ((threadIdx.x & 31) == 0) red[turn][threadIdx.x >> 5] = st;
        __syncthreads();
        if (threadIdx.x == 0) {
            Stat all = red[turn][0];
            for (int w = 1; w < 8; w++) all = join(all, red[turn][w]);
            const Sums s = finish_row(q, p, r, all);
            sums.loss += s.loss, sums.count += s.count;
        }
        turn ^= 1;
    }
    if (p.loss) finish_loss(p, sums, part, counter);
}

// Sums of a pair's two sequences, the pair's loss term and its sequences' factors; the last block sums the terms.
__global__ void __launch_bounds__(256) k_pairs(nck_pairs p, const double *__restrict__ lp, double *term, unsigned *counter) {
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
        term[i] = (1.0 - eps) * (soft + (h < 0.0 ? -h : 0.0)) + eps * (soft + (h > 0.0 ? h : 0.0));
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

// The gradient of one row by a team of W threads: dst (+)= c (1[j = a] - exp(z - m) inv).
template <int W, int U, bool ACC>
__device__ __forceinline__ void grad_row(const float *z, float *dst, int64_t V, float c, float m, float inv, int64_t a, int t) {
    if (c == 0.0f) { // nothing of the row is read
        if (ACC) return;
        const int64_t lead = lead_of(dst, V), nv = (V - lead) >> 2, tail = lead + 4 * nv;
        float4 *d4 = reinterpret_cast<float4 *>(dst + lead);
        for (int64_t i = t; i < nv; i += W) d4[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (t < lead) dst[t] = 0.0f;
        if (t < V - tail) dst[tail + t] = 0.0f;
        return;
    }
    const float f = -c * inv;
    const auto one = [&](int64_t j) {
        float v = f * __expf(z[j] - m);
        if (j == a) v += c;
        dst[j] = ACC ? dst[j] + v : v;
    };
    if ((((uintptr_t)z ^ (uintptr_t)dst) & 15) != 0) { // rows of another alignment than their gradient's
        for (int64_t j = t; j < V; j += W) one(j);
        return;
    }
    const int64_t lead = lead_of(z, V), nv = (V - lead) >> 2, tail = lead + 4 * nv;
    const float4 *z4 = reinterpret_cast<const float4 *>(z + lead);
    float4 *d4 = reinterpret_cast<float4 *>(dst + lead);
    for (int64_t i = t; i < nv; i += W * U) {
        float4 v[U], old[ACC ? U : 1];
#pragma unroll
        for (int u = 0; u < U; u++)
            if (i + u * W < nv) {
                v[u] = __ldg(z4 + i + u * W);
                if (ACC) old[ACC ? u : 0] = d4[i + u * W];
            }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (i + u * W >= nv) break;
            float4 g = make_float4(f * __expf(v[u].x - m), f * __expf(v[u].y - m), f * __expf(v[u].z - m), f * __expf(v[u].w - m));
            const uint64_t k = (uint64_t)(a - lead - 4 * (i + u * W));
            if (k < 4) g.x += k == 0 ? c : 0.0f, g.y += k == 1 ? c : 0.0f, g.z += k == 2 ? c : 0.0f, g.w += k == 3 ? c : 0.0f;
            if (ACC) {
                const float4 o = old[ACC ? u : 0];
                g.x += o.x, g.y += o.y, g.z += o.z, g.w += o.w;
            }
            d4[i + u * W] = g;
        }
    }
    if (t < lead) one(t);
    if (t < V - tail) one(tail + t);
}

template <int W, bool ACC>
__global__ void __launch_bounds__(256) k_rows_grad(nck_rows q, nck_rows_grad g) {
    const int t = threadIdx.x % W;
    const float up = g.up[0] * (g.scale ? g.scale[0] : 1.0f);
    const int64_t teams = (int64_t)gridDim.x * (256 / W);
    for (int64_t r = (int64_t)blockIdx.x * (256 / W) + threadIdx.x / W; r < q.N; r += teams) {
        const float c = counted(q, r) ? up * g.coef[r / g.per_coef] : 0.0f;
        const float2 st = c == 0.0f ? make_float2(0.f, 0.f) : reinterpret_cast<const float2 *>(q.stat)[r];
        int64_t a = q.lab[r];
        if (a < 0 || a >= q.V) a = 0;
        grad_row<W, W == 32 ? 1 : 4, ACC>(row_of(q, r), g.dz + r * q.V, q.V, c, st.x, st.y, a, t);
    }
}

int blocks_for(const nck_dev *d, int64_t want, int per_sm) {
    const int64_t room = (int64_t)(d->sm_count > 0 ? d->sm_count : 148) * per_sm;
    return (int)(want < 1 ? 1 : want < room ? want : room);
}

}  // namespace

extern "C" void nck_rows_logp(nck_dev *d, const nck_rows *q, const nck_policy *p) {
    nck_rows rows = *q;
    rows.status = d->status;
    nck_policy pol;
    if (p) pol = *p;
    else pol = nck_policy{};
    Scope sc(d, "logits_logp", 4.0 * q->N * q->V, 4.0 * q->N * q->V);
    double2 *part = (double2 *)d->scratch;
    if (q->V <= kWarpRow) {
        const int room = (d->sm_count > 0 ? d->sm_count : 148) * 64;  // warps of a full GPU
        int64_t run = (q->N + room - 1) / room;
        run = run < 1 ? 1 : run > 32 ? 32 : run;
        k_rows_warp<<<blocks_for(d, (q->N + run * 8 - 1) / (run * 8), 8), 256, 0, NCK_STREAM(d)>>>(rows, pol, (int)run, part,
                                                                                                d->counters);
    } else {
        k_rows_block<<<blocks_for(d, q->N, 8), 256, 0, NCK_STREAM(d)>>>(rows, pol, part, d->counters);
    }
    NCK_LAUNCHED(d, 1);
}

extern "C" void nck_pref_pairs(nck_dev *d, const nck_pairs *p, const double *lp) {
    Scope sc(d, "preference_pairs", 0.0, 16.0 * p->P * p->T);
    k_pairs<<<(unsigned)p->P, 256, 0, NCK_STREAM(d)>>>(*p, lp, p->term, d->counters);
    NCK_LAUNCHED(d, 1);
}

extern "C" void nck_rows_bwd(nck_dev *d, const nck_rows *q, const nck_rows_grad *g) {
    if (q->N == 0) return;
    Scope sc(d, "logits_logp_bwd", 4.0 * q->N * q->V, 8.0 * q->N * q->V);
    if (q->V <= kWarpRow) {
        const int grid = blocks_for(d, (q->N + 7) / 8, 16);
        if (g->acc) k_rows_grad<32, true><<<grid, 256, 0, NCK_STREAM(d)>>>(*q, *g);
        else k_rows_grad<32, false><<<grid, 256, 0, NCK_STREAM(d)>>>(*q, *g);
    } else {
        const int grid = blocks_for(d, q->N, 16);
        if (g->acc) k_rows_grad<256, true><<<grid, 256, 0, NCK_STREAM(d)>>>(*q, *g);
        else k_rows_grad<256, false><<<grid, 256, 0, NCK_STREAM(d)>>>(*q, *g);
    }
    NCK_LAUNCHED(d, 1);
}
