// Query/key head norms and rotary positions in one pass, forward and backward.
//
//   r = (mean_d x_d^2 + eps)^-1/2,  n = x r,  u = n w          (w: the query or the key weight, by head)
//   pair (a, b) of u turned by its angle: y_a = u_a cos - u_b sin,  y_b = u_b cos + u_a sin
// and, with g = the inverse turn of dy:
//   dw = sum over rows of g n,   dx = r (g w - n mean_d(g w n))
//
// Both passes are bound by HBM: x read and y written (8 bytes an element) forward, x and dy read and dx
// written (12 bytes) backward, about ten operations an element. A row (one head of one token) belongs to a
// group of 1 to 32 lanes, each owning up to four pairs as two vector loads, so the norm is a few shuffles and
// the rotation needs no exchange between lanes. A group walks heads of one token, so a lane computes the sines
// and cosines of its own pairs once a token and keeps them in registers: no table in memory, no barrier. The
// angle is reduced in 64 bits (position times turns per step, minus its nearest whole number): positions of a
// million lose no digits, and the reduced turn, at most one half, is exact to 2^-26 in 32 bits.
#include "k_common.cuh"

using namespace nck;

namespace {

constexpr int kMaxOwn = 4;  // pairs per lane

__device__ __forceinline__ void load(const float *p, float (&v)[1]) { v[0] = *p; }
__device__ __forceinline__ void load(const float *p, float (&v)[2]) {
    const float2 u = *reinterpret_cast<const float2 *>(p);
    v[0] = u.x, v[1] = u.y;
}
__device__ __forceinline__ void load(const float *p, float (&v)[4]) {
    const float4 u = *reinterpret_cast<const float4 *>(p);
    v[0] = u.x, v[1] = u.y, v[2] = u.z, v[3] = u.w;
}

__device__ __forceinline__ void store(float *p, const float (&v)[1]) { *p = v[0]; }
__device__ __forceinline__ void store(float *p, const float (&v)[2]) {
    *reinterpret_cast<float2 *>(p) = make_float2(v[0], v[1]);
}
__device__ __forceinline__ void store(float *p, const float (&v)[4]) {
    *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
}

// How the groups share the work: lanes per group, heads per item, items = tokens x chunks of heads.
struct RopeGrid {
    int lpr, per_item;
    int64_t chunks, items;
};

// The pairs of one row that a lane owns, NJ vectors of VEC pairs: the first and second elements of each
// pair. Pairs behind the row's end read as zero.
template <int VEC, int NJ>
struct Own {
    float a[NJ * VEC], b[NJ * VEC];
    template <bool INTER>
    __device__ __forceinline__ void get(const float *row, int half, int lpr, int l) {
#pragma unroll
        for (int j = 0; j < NJ; j++) {
            const int p = (j * lpr + l) * VEC;
            float u[VEC], v[VEC];
#pragma unroll
            for (int i = 0; i < VEC; i++) u[i] = v[i] = 0.0f;
            if (p < half) {
                load(row + (INTER ? 2 * p : p), u);
                load(row + (INTER ? 2 * p + VEC : half + p), v);
            }
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                if (INTER) { // u, v hold 2 VEC neighbours: pair i is elements 2i and 2i + 1
                    a[j * VEC + i] = 2 * i < VEC ? u[(2 * i) % VEC] : v[(2 * i) % VEC];
                    b[j * VEC + i] = 2 * i + 1 < VEC ? u[(2 * i + 1) % VEC] : v[(2 * i + 1) % VEC];
                } else {
                    a[j * VEC + i] = u[i];
                    b[j * VEC + i] = v[i];
                }
            }
        }
    }
    template <bool INTER>
    __device__ __forceinline__ void put(float *row, int half, int lpr, int l) const {
#pragma unroll
        for (int j = 0; j < NJ; j++) {
            const int p = (j * lpr + l) * VEC;
            if (p >= half) continue;
            float u[VEC], v[VEC];
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                if (INTER) {
                    const int e = i, f = VEC + i; // elements e of u, f of the 2 VEC neighbours
                    u[i] = e % 2 ? b[j * VEC + e / 2] : a[j * VEC + e / 2];
                    v[i] = f % 2 ? b[j * VEC + f / 2] : a[j * VEC + f / 2];
                } else {
                    u[i] = a[j * VEC + i];
                    v[i] = b[j * VEC + i];
                }
            }
            store(row + (INTER ? 2 * p : p), u);
            store(row + (INTER ? 2 * p + VEC : half + p), v);
        }
    }
};

__device__ __forceinline__ float group_sum(float v, int lpr, unsigned mask) {
    for (int o = lpr >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(mask, v, o);
    return v;
}

// cos and sin of the lane's pairs at one token
template <int N>
__device__ __forceinline__ void turn_of(const nck_rope &q, int64_t b, int64_t t, const double (&turns)[N],
                                        const int (&axis)[N], float (&c)[N], float (&s)[N]) {
    int at[3] = {0, 0, 0};
    if (q.pos) {
        const int32_t *p = q.pos + b * q.pos_b + t * q.pos_t;
        at[0] = p[0];
        if (q.n_axes > 1) at[1] = p[1];
        if (q.n_axes > 2) at[2] = p[2];
    } else {
        at[0] = (int)t;
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
        const double full = (double)(axis[i] == 0 ? at[0] : axis[i] == 1 ? at[1] : at[2]) * turns[i];
        sincospif(2.0f * (float)(full - rint(full)), &s[i], &c[i]);
    }
}

template <int VEC, int NJ>
__device__ __forceinline__ void own_turns(const nck_rope &q, int half, int lpr, int l, double (&turns)[NJ * VEC],
                                          int (&axis)[NJ * VEC]) {
#pragma unroll
    for (int j = 0; j < NJ; j++)
#pragma unroll
        for (int i = 0; i < VEC; i++) {
            const int p = (j * lpr + l) * VEC + i;
            turns[j * VEC + i] = p < half ? q.turns[p] : 0.0;
            axis[j * VEC + i] = p < half ? q.axis[p] : 0;
        }
}

template <int VEC, int NJ, bool INTER>
__global__ void __launch_bounds__(256) k_rope_fwd(const __grid_constant__ nck_rope q, RopeGrid g, float *__restrict__ y) {
    constexpr int N = VEC * NJ, U = 2; // U rows in flight
    const int lane = threadIdx.x & 31, l = threadIdx.x & (g.lpr - 1), half = q.D >> 1;
    const unsigned mask = g.lpr == 32 ? 0xffffffffu : ((1u << g.lpr) - 1u) << (lane & ~(g.lpr - 1));
    const int64_t groups = (int64_t)gridDim.x * (blockDim.x / g.lpr);
    const float inv_d = 1.0f / (float)q.D;
    double turns[N];
    int axis[N];
    own_turns<VEC, NJ>(q, half, g.lpr, l, turns, axis);
    for (int64_t it = (int64_t)blockIdx.x * (blockDim.x / g.lpr) + threadIdx.x / g.lpr; it < g.items; it += groups) {
        const int64_t tok = it / g.chunks, b = tok / q.T, t = tok - b * q.T;
        const int h0 = (int)(it - tok * g.chunks) * g.per_item, h1 = min(h0 + g.per_item, q.H);
        const float *x = q.x + b * q.sb + t * q.st;
        float *out = y + tok * q.H * q.D;
        float c[N], s[N];
        turn_of<N>(q, b, t, turns, axis, c, s);
        for (int h = h0; h < h1; h += U) {
            Own<VEC, NJ> row[U];
#pragma unroll
            for (int k = 0; k < U; k++)
                if (h + k < h1) row[k].template get<INTER>(x + (h + k) * q.sh, half, g.lpr, l);
#pragma unroll
            for (int k = 0; k < U; k++) {
                if (h + k >= h1) break;
                Own<VEC, NJ> &v = row[k];
                if (q.norm) {
                    float ss = 0.0f;
#pragma unroll
                    for (int i = 0; i < N; i++) ss = fmaf(v.a[i], v.a[i], fmaf(v.b[i], v.b[i], ss));
                    const float r = rsqrtf(fmaf(group_sum(ss, g.lpr, mask), inv_d, q.eps));
#pragma unroll
                    for (int i = 0; i < N; i++) v.a[i] *= r, v.b[i] *= r;
                }
                if (const float *w = h + k < q.HQ ? q.wq : q.wk) {
                    Own<VEC, NJ> ws;
                    ws.template get<INTER>(w, half, g.lpr, l);
#pragma unroll
                    for (int i = 0; i < N; i++) v.a[i] *= ws.a[i], v.b[i] *= ws.b[i];
                }
#pragma unroll
                for (int i = 0; i < N; i++) {
                    const float ua = v.a[i], ub = v.b[i];
                    v.a[i] = fmaf(ua, c[i], -(ub * s[i]));
                    v.b[i] = fmaf(ub, c[i], ua * s[i]);
                }
                v.template put<INTER>(out + (int64_t)(h + k) * q.D, half, g.lpr, l);
            }
        }
    }
}

// part (may be NULL): the block's sums of g n over its query rows and over its key rows, [block][2][D]
template <int VEC, int NJ, bool INTER>
__global__ void __launch_bounds__(256) k_rope_bwd(const __grid_constant__ nck_rope q, RopeGrid g,
                                                  const float *__restrict__ dy, float *dx, int acc,
                                                  float *__restrict__ part) {
    constexpr int N = VEC * NJ;
    __shared__ float red[256 * 2 * kMaxOwn];
    const int lane = threadIdx.x & 31, l = threadIdx.x & (g.lpr - 1), half = q.D >> 1;
    const unsigned mask = g.lpr == 32 ? 0xffffffffu : ((1u << g.lpr) - 1u) << (lane & ~(g.lpr - 1));
    const int per_block = blockDim.x / g.lpr, mine = threadIdx.x / g.lpr;
    const int64_t groups = (int64_t)gridDim.x * per_block;
    const float inv_d = 1.0f / (float)q.D;
    double turns[N];
    int axis[N];
    own_turns<VEC, NJ>(q, half, g.lpr, l, turns, axis);
    Own<VEC, NJ> sum[2];
#pragma unroll
    for (int i = 0; i < N; i++) sum[0].a[i] = sum[0].b[i] = sum[1].a[i] = sum[1].b[i] = 0.0f;
    for (int64_t it = (int64_t)blockIdx.x * per_block + mine; it < g.items; it += groups) {
        const int64_t tok = it / g.chunks, b = tok / q.T, t = tok - b * q.T;
        const int h0 = (int)(it - tok * g.chunks) * g.per_item, h1 = min(h0 + g.per_item, q.H);
        const float *x = q.x + b * q.sb + t * q.st;
        float c[N], s[N];
        turn_of<N>(q, b, t, turns, axis, c, s);
        for (int h = h0; h < h1; h++) {
            const int64_t at = (tok * q.H + h) * q.D;
            Own<VEC, NJ> v, d;
            v.template get<INTER>(x + h * q.sh, half, g.lpr, l);
            d.template get<INTER>(dy + at, half, g.lpr, l);
            float r = 1.0f;
            if (q.norm) {
                float ss = 0.0f;
#pragma unroll
                for (int i = 0; i < N; i++) ss = fmaf(v.a[i], v.a[i], fmaf(v.b[i], v.b[i], ss));
                r = rsqrtf(fmaf(group_sum(ss, g.lpr, mask), inv_d, q.eps));
            }
#pragma unroll
            for (int i = 0; i < N; i++) {
                const float ya = d.a[i], yb = d.b[i];
                d.a[i] = fmaf(ya, c[i], yb * s[i]);
                d.b[i] = fmaf(yb, c[i], -(ya * s[i]));
                v.a[i] *= r, v.b[i] *= r; // n
            }
            if (part) {
                const bool query = h < q.HQ;
#pragma unroll
                for (int i = 0; i < N; i++) {
                    const float ga = d.a[i] * v.a[i], gb = d.b[i] * v.b[i];
                    sum[0].a[i] += query ? ga : 0.0f, sum[0].b[i] += query ? gb : 0.0f;
                    sum[1].a[i] += query ? 0.0f : ga, sum[1].b[i] += query ? 0.0f : gb;
                }
            }
            if (!dx) continue;
            if (const float *w = h < q.HQ ? q.wq : q.wk) {
                Own<VEC, NJ> ws;
                ws.template get<INTER>(w, half, g.lpr, l);
#pragma unroll
                for (int i = 0; i < N; i++) d.a[i] *= ws.a[i], d.b[i] *= ws.b[i];
            }
            if (q.norm) {
                float dot = 0.0f;
#pragma unroll
                for (int i = 0; i < N; i++) dot = fmaf(d.a[i], v.a[i], fmaf(d.b[i], v.b[i], dot));
                const float m = group_sum(dot, g.lpr, mask) * inv_d;
#pragma unroll
                for (int i = 0; i < N; i++) {
                    d.a[i] = r * fmaf(-m, v.a[i], d.a[i]);
                    d.b[i] = r * fmaf(-m, v.b[i], d.b[i]);
                }
            }
            if (acc) {
                Own<VEC, NJ> old;
                old.template get<INTER>(dx + at, half, g.lpr, l);
#pragma unroll
                for (int i = 0; i < N; i++) d.a[i] += old.a[i], d.b[i] += old.b[i];
            }
            d.template put<INTER>(dx + at, half, g.lpr, l);
        }
    }
    if (!part) return;
    for (int k = 0; k < 2; k++) {
        __syncthreads();
        sum[k].template put<INTER>(red + mine * q.D, half, g.lpr, l);
        __syncthreads();
        for (int d = threadIdx.x; d < q.D; d += blockDim.x) {
            float t = 0.0f;
            for (int j = 0; j < per_block; j++) t += red[j * q.D + d];
            part[((int64_t)blockIdx.x * 2 + k) * q.D + d] = t;
        }
    }
}

// dw (+)= the blocks' partial sums, in block order; 32 columns a block, 8 slices of the blocks each
__global__ void __launch_bounds__(256) k_rope_dw(const float *__restrict__ part, int blocks, int D, float *dwq, int acc_q,
                                                 float *dwk, int acc_k) {
    __shared__ double red[8][32];
    const int col = blockIdx.x * 32 + (threadIdx.x & 31), sl = threadIdx.x >> 5;
    double t = 0.0;
    if (col < 2 * D)
        for (int b = sl; b < blocks; b += 8) t += (double)part[(int64_t)b * 2 * D + col];
    red[sl][threadIdx.x & 31] = t;
    __syncthreads();
    if (sl || col >= 2 * D) return;
    for (int j = 1; j < 8; j++) t += red[j][threadIdx.x];
    float *dw = col < D ? dwq : dwk;
    if (!dw) return;
    float *to = dw + (col < D ? col : col - D);
    const bool acc = col < D ? acc_q : acc_k;
    *to = acc ? *to + (float)t : (float)t;
}

bool aligned(const void *p, int vec) { return ((uintptr_t)p & (size_t)(4 * vec - 1)) == 0; }

// The widest vector that x's layout and every pointer of the pass allow: 4, 2 or 1 pairs.
int vector_of(const nck_rope *q, const void *p1, const void *p2) {
    for (int vec = 4; vec > 1; vec >>= 1) {
        bool ok = q->D % (2 * vec) == 0 && aligned(q->x, vec) && aligned(q->wq, vec) && aligned(q->wk, vec) &&
                  aligned(p1, vec) && aligned(p2, vec);
        ok = ok && (q->B == 1 || q->sb % vec == 0) && (q->T == 1 || q->st % vec == 0) && (q->H == 1 || q->sh % vec == 0);
        if (ok) return vec;
    }
    return 1;
}

// Groups of the smallest power of two lanes that holds a row, whole tokens per group when there are enough
// tokens to fill the GPU, fewer heads per group (each repeats the token's angles) when there are not.
RopeGrid split_of(const nck_dev *d, const nck_rope *q, int vec) {
    RopeGrid g;
    const int vecs = (q->D / 2 + vec - 1) / vec;
    g.lpr = 1;
    while (g.lpr < vecs && g.lpr < 32) g.lpr <<= 1;
    const int64_t tokens = q->B * q->T, room = (int64_t)d->sm_count * 2048 / g.lpr;
    int64_t per = tokens * q->H / room;
    if (per < 1) per = 1;
    if (per > q->H) per = q->H;
    g.per_item = (int)per;
    g.chunks = (q->H + per - 1) / per;
    g.items = tokens * g.chunks;
    return g;
}

template <int VEC, int NJ>
void launch_fwd(nck_dev *d, const nck_rope *q, const RopeGrid &g, float *y) {
    const int64_t blocks = (g.items * g.lpr + 255) / 256;
    const int grid = (int)(blocks < ((int64_t)1 << 30) ? blocks : (int64_t)1 << 30);
    if (q->interleaved) k_rope_fwd<VEC, NJ, true><<<grid, 256, 0, NCK_STREAM(d)>>>(*q, g, y);
    else k_rope_fwd<VEC, NJ, false><<<grid, 256, 0, NCK_STREAM(d)>>>(*q, g, y);
    NCK_LAUNCHED(d, 1);
}

template <int VEC, int NJ, bool INTER>
int launch_bwd(nck_dev *d, const nck_rope *q, const RopeGrid &g, const float *dy, float *dx, int acc, float *part) {
    static int room = 0;
    if (!room) room = resident_blocks(d, k_rope_bwd<VEC, NJ, INTER>, 256);
    const int64_t blocks = (g.items * g.lpr + 255) / 256;
    const int grid = (int)(blocks < room ? blocks : room);
    k_rope_bwd<VEC, NJ, INTER><<<grid, 256, 0, NCK_STREAM(d)>>>(*q, g, dy, dx, acc, part);
    NCK_LAUNCHED(d, 1);
    return grid;
}

}  // namespace

extern "C" void nck_rope_fwd(nck_dev *d, const nck_rope *q, float *y) {
    const double n = (double)q->B * q->T * q->H * q->D;
    if (n == 0) return;
    Scope sc(d, "qk_norm_rope", 10.0 * n, 8.0 * n);
    const int vec = vector_of(q, y, nullptr);
    const RopeGrid g = split_of(d, q, vec);
    if (vec == 4) launch_fwd<4, 1>(d, q, g, y);
    else if (vec == 2) launch_fwd<2, 2>(d, q, g, y);
    else launch_fwd<1, 4>(d, q, g, y);
}

extern "C" void nck_rope_bwd(nck_dev *d, const nck_rope *q, const float *dy, float *dx, int acc_x, float *dwq, int acc_q,
                             float *dwk, int acc_k) {
    const double n = (double)q->B * q->T * q->H * q->D;
    Scope sc(d, "qk_norm_rope_bwd", 20.0 * n, 12.0 * n);
    float *part = dwq || dwk ? (float *)d->scratch : nullptr;
    int grid = 0;
    if (n > 0 && (dx || part)) {
        const int vec = vector_of(q, dy, dx);
        const RopeGrid g = split_of(d, q, vec);
        if (vec == 4)
            grid = q->interleaved ? launch_bwd<4, 1, true>(d, q, g, dy, dx, acc_x, part)
                                  : launch_bwd<4, 1, false>(d, q, g, dy, dx, acc_x, part);
        else if (vec == 2)
            grid = q->interleaved ? launch_bwd<2, 2, true>(d, q, g, dy, dx, acc_x, part)
                                  : launch_bwd<2, 2, false>(d, q, g, dy, dx, acc_x, part);
        else
            grid = q->interleaved ? launch_bwd<1, 4, true>(d, q, g, dy, dx, acc_x, part)
                                  : launch_bwd<1, 4, false>(d, q, g, dy, dx, acc_x, part);
    }
    if (!part) return;
    k_rope_dw<<<(2 * q->D + 31) / 32, 256, 0, NCK_STREAM(d)>>>(part, grid, q->D, dwq, acc_q, dwk, acc_k);
    NCK_LAUNCHED(d, 1);
}
