// Query/key head norms and rotary positions in one pass, forward and backward.
//
//   r = (mean_d x_d^2 + eps)^-1/2,  n = x r,  u = n w          (w: the query or the key weight, by head)
//   pair (a, b) of u turned by its angle: y_a = u_a cos - u_b sin,  y_b = u_b cos + u_a sin
// and, with g = the inverse turn of dy:
//   dw = sum over rows of g n,   dx = r (g w - n mean_d(g w n))
//
// Both passes are bound by HBM: x read and y written (8 bytes an element) forward, x and dy read and dx
// written (12 bytes) backward, about ten operations an element. A row (one head of one token) belongs to a
// group of LPR lanes (1 to 32), each owning up to four pairs as two vector loads, so the norm is a few
// shuffles and the rotation needs no exchange between lanes. A warp takes the same run of heads of 32 / LPR
// tokens, all lanes in step, so a lane forms the sines and cosines of its own pairs once a token and run,
// multiplies them by the weights once, and keeps them in registers: no table in memory, no barrier. Warps walk
// a grid of one full wave. A group need not be a power of two of lanes: three heads of 72 or 80 share a
// warp on nine or ten lanes each, where two on sixteen would leave half the issue slots idle (24 x 1369 x 24 heads
// of 72: 88 instead of 102 us; 4 x 8000 x 16 heads of 66 69 instead of 131).
//
// Angles are formed in whole numbers: a pair's turns per step are kept as a 64-bit fraction of a turn, a
// position times it modulo 2^64 is the fraction of the turn reached, and its upper half (cut off below 2^-32 turns)
// splits into quarter turns and a remainder of at most 1/8 turn. The steps are off by 9 units of 2^-64 at most for
// bases above 1 (3 for 10000; ops_rope.c), so the angle is by 2^-32 + |position| 9 * 2^-64 turns: below 2^-29 at any i32
// position, a fifth of 2^-24 in radians. On that range sine and cosine are polynomials (interpolation in the remainder's
// square at Chebyshev nodes), off by less than 1.9 * 2^-24 with the rounding of the remainder.
#include "k_common.cuh"

using namespace nck;

namespace {

// the arithmetic of two pairs
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return make_float2(fmaf(a.x, b.x, c.x), fmaf(a.y, b.y, c.y)); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return make_float2(a.x * b.x, a.y * b.y); }
__device__ __forceinline__ float2 neg2(float2 a) { return make_float2(-a.x, -a.y); }
__device__ __forceinline__ float2 both(float f) { return make_float2(f, f); }

template <int VEC>
__device__ __forceinline__ void load(const float *p, float (&v)[VEC]) {
    if constexpr (VEC == 1) {
        v[0] = *p;
    } else if constexpr (VEC == 2) {
        const float2 u = *reinterpret_cast<const float2 *>(p);
        v[0] = u.x, v[1] = u.y;
    } else {
        const float4 u = *reinterpret_cast<const float4 *>(p);
        v[0] = u.x, v[1] = u.y, v[2] = u.z, v[3] = u.w;
    }
}

template <int VEC>
__device__ __forceinline__ void store(float *p, const float (&v)[VEC]) {
    if constexpr (VEC == 1) *p = v[0];
    else if constexpr (VEC == 2) *reinterpret_cast<float2 *>(p) = make_float2(v[0], v[1]);
    else *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
}

// How warps share the work: an item is `run` heads of the 32 / LPR tokens of a tile.
struct RopeGrid {
    int run, tiles;          // tiles of tokens
    int64_t items;
    FastDiv by_tiles, by_T;
};

constexpr int kOwn = 4, kTwo = kOwn / 2; // pairs per lane, and their register pairs

// Rows that a lane has in flight, two blocks of 256 threads an SM (128 registers a thread); narrower vectors have more
// addresses a row and take a row less. More blocks of fewer rows keep less in flight for the same registers. Forward at
// 4 x 4680 x 24 heads of 128: 78 us with 4 rows (70 at the copy rate), 79 with 3, 80.5 with 6, 85 with 8, and 82 to 84
// with 3 or 4 blocks of 2; 24 x 1369 x 24 heads of 72: 89, 95, 84, 85 and 88 us (69 at the copy rate); 4 x 8000 x 16
// heads of 64 50, 53, 51 and 52 us (41). Backward at the first: 118 us with 2 rows (105 at the copy rate), 132 with
// 3 blocks of 1, 130 with 3 rows.
constexpr int kRowsFwd = 4, kRowsBwd = 2;

// Pairs in a lane's vector of VEC floats (two of them for split halves; with neighbours one vector holds both
// elements of its pairs, and a float of its own is half a pair).
template <int VEC, bool INTER>
constexpr int kPairs = INTER ? (VEC > 1 ? VEC / 2 : 1) : VEC;

// The pairs of one row that a lane owns, kOwn / kPairs vectors' worth: the first and the second elements of each pair.
// Neighbouring lanes' vectors are neighbours, so that a load or store of a warp covers whole sectors. Neighbours as
// pairs need sizes that are multiples of 4 only for float4 (two vectors a lane, 16 bytes apart, wrote each sector twice
// and needed multiples of 8: forward 16 x 4000 x 16 heads of 20 57 us, now 40; both passes of 4 x 8000 x 8 heads of 100
// 129 us, now 110; 24 x 1369 x 24 heads of 72 86 us, now 84.5).
// Pairs behind the row's end read as zero.
template <int VEC, int LPR, bool INTER>
struct Own {
    float2 a[kTwo], b[kTwo];
    static constexpr int P = kPairs<VEC, INTER>, NJ = kOwn / P;
    __device__ __forceinline__ void get(const float *row, int half, int l) {
        float x[kOwn], y[kOwn];
#pragma unroll
        for (int j = 0; j < NJ; j++) {
            const int p = (j * LPR + l) * P;
            if constexpr (INTER) {
                float u[2 * P] = {};
                if (p < half) {
                    if constexpr (VEC == 1) u[0] = row[2 * p], u[1] = row[2 * p + 1];
                    else load<2 * P>(row + 2 * p, u);
                }
#pragma unroll
                for (int i = 0; i < P; i++) x[j * P + i] = u[2 * i], y[j * P + i] = u[2 * i + 1];
            } else {
                float u[P] = {}, v[P] = {};
                if (p < half) {
                    load<P>(row + p, u);
                    load<P>(row + half + p, v);
                }
#pragma unroll
                for (int i = 0; i < P; i++) x[j * P + i] = u[i], y[j * P + i] = v[i];
            }
        }
#pragma unroll
        for (int i = 0; i < kTwo; i++) a[i] = make_float2(x[2 * i], x[2 * i + 1]), b[i] = make_float2(y[2 * i], y[2 * i + 1]);
    }
    __device__ __forceinline__ void put(float *row, int half, int l) const {
        const float x[kOwn] = {a[0].x, a[0].y, a[1].x, a[1].y}, y[kOwn] = {b[0].x, b[0].y, b[1].x, b[1].y};
#pragma unroll
        for (int j = 0; j < NJ; j++) {
            const int p = (j * LPR + l) * P;
            if (p >= half) continue;
            if constexpr (INTER) {
                float u[2 * P];
#pragma unroll
                for (int i = 0; i < P; i++) u[2 * i] = x[j * P + i], u[2 * i + 1] = y[j * P + i];
                if constexpr (VEC == 1) row[2 * p] = u[0], row[2 * p + 1] = u[1];
                else store<2 * P>(row + 2 * p, u);
            } else {
                float u[P], v[P];
#pragma unroll
                for (int i = 0; i < P; i++) u[i] = x[j * P + i], v[i] = y[j * P + i];
                store<P>(row + p, u);
                store<P>(row + half + p, v);
            }
        }
    }
    __device__ __forceinline__ void fill(float f) {
#pragma unroll
        for (int i = 0; i < kTwo; i++) a[i] = b[i] = both(f);
    }
};

// The sum over a group's lanes, in all of them. Lanes behind the last whole group get some number.
template <int LPR>
__device__ __forceinline__ float group_sum(float v, int lane, int l) {
    if constexpr ((LPR & (LPR - 1)) == 0) {
#pragma unroll
        for (int o = LPR >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
        return v;
    } else {
        constexpr int kTop = LPR > 8 ? 8 : LPR > 4 ? 4 : 2;
#pragma unroll
        for (int o = kTop; o > 0; o >>= 1) {
            const float u = __shfl_down_sync(~0u, v, o);
            if (l < o && l + o < LPR) v += u;
        }
        return __shfl_sync(~0u, v, lane - l);
    }
}

__device__ __forceinline__ float sum2(float2 s) { return s.x + s.y; }

// The pairs' fractions of a turn per step and their axes, in shared memory: registers are better spent on rows in
// flight, and the parameters' constant bank serves one address at a time.
struct Turns {
    uint64_t step[NCK_ROPE_MAX_DIM / 2];
    int axis[NCK_ROPE_MAX_DIM / 2];
    __device__ __forceinline__ void fill(const nck_rope &q) {
        for (int p = threadIdx.x; p < NCK_ROPE_MAX_DIM / 2; p += blockDim.x) step[p] = q.turns[p], axis[p] = q.axis[p];
        __syncthreads();
    }
    // cos and sin of the lane's pairs at token (b, t)
    template <int P, int LPR>
    __device__ __forceinline__ void at(const nck_rope &q, int64_t b, int64_t t, int l, float2 (&c)[kTwo], float2 (&s)[kTwo]) const {
        int pos[3] = {(int)t, 0, 0};
        if (q.pos) {
            const int32_t *p = q.pos + b * q.pos_b + t * q.pos_t;
            pos[0] = p[0];
            if (q.n_axes > 1) pos[1] = p[1];
            if (q.n_axes > 2) pos[2] = p[2];
        }
        float cv[kOwn], sv[kOwn];
#pragma unroll
        for (int i = 0; i < kOwn; i++) {
            const int p = ((i / P * LPR + l) * P + i % P) & (NCK_ROPE_MAX_DIM / 2 - 1); // (behind the row: any)
            const int a = axis[p];
            const int64_t at = a == 0 ? pos[0] : a == 1 ? pos[1] : pos[2];
            const int32_t turn = (int32_t)(((uint64_t)at * step[p]) >> 32);   // of 2^32
            const uint32_t quarter = ((uint32_t)turn + (1u << 29)) >> 30;
            const float g = (float)(int32_t)((uint32_t)turn - (quarter << 30)) * 2.3283064365386963e-10f, g2 = g * g;
            const float sn = g * fmaf(g2, fmaf(g2, fmaf(g2, -75.401611f, 81.592545f), -41.341663f), 6.2831855f);
            const float cs = fmaf(g2, fmaf(g2, fmaf(g2, -83.591820f, 64.921234f), -19.739153f), 1.0f);
            const float x = quarter & 1 ? sn : cs, y = quarter & 1 ? cs : sn;
            cv[i] = (quarter + 1) & 2 ? -x : x;
            sv[i] = quarter & 2 ? -y : y;
        }
#pragma unroll
        for (int i = 0; i < kTwo; i++) c[i] = make_float2(cv[2 * i], cv[2 * i + 1]), s[i] = make_float2(sv[2 * i], sv[2 * i + 1]);
    }
};

// An item's heads [h0, h1), the lane's token (live: it exists; a lane without one reads the last token).
template <int LPR>
struct Item {
    int h0, h1, tok, b, t;
    bool live;
    __device__ __forceinline__ Item(const nck_rope &q, const RopeGrid &g, int64_t it, int sub) {
        constexpr int per = 32 / LPR;
        const uint32_t k = (uint32_t)it, chunk = g.by_tiles.div(k);
        h0 = (int)chunk * g.run;
        h1 = min(h0 + g.run, q.H);
        const int64_t at = (int64_t)(k - chunk * (uint32_t)g.tiles) * per + sub, tokens = q.B * q.T;
        live = sub < per && at < tokens;
        tok = (int)(at < tokens ? at : tokens - 1);
        b = (int)g.by_T.div((uint32_t)tok);
        t = tok - b * (int)q.T;
    }
};

template <int VEC, int LPR, bool INTER>
__global__ void __launch_bounds__(256, 2) k_rope_fwd(const __grid_constant__ nck_rope q, const RopeGrid g, float *__restrict__ y) {
    constexpr int U = VEC == 4 ? kRowsFwd : kRowsFwd - 1;
    typedef Own<VEC, LPR, INTER> Row;
    const int lane = threadIdx.x & 31, l = lane % LPR, half = q.D >> 1;
    const float inv_d = 1.0f / (float)q.D;
    __shared__ Turns turns;
    turns.fill(q);
    cudaGridDependencySynchronize();
    for (int64_t it = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); it < g.items; it += (int64_t)gridDim.x * 8) {
        const Item<LPR> m(q, g, it, lane / LPR);
        const float *x = q.x + m.b * q.sb + m.t * q.st + m.h0 * q.sh;
        float *out = y + ((int64_t)m.tok * q.H + m.h0) * q.D;
        Row row[U]; // the first rows are on their way while the angles are formed
#pragma unroll
        for (int k = 0; k < U; k++)
            if (m.h0 + k < m.h1) row[k].get(x + k * q.sh, half, l);
        float2 c[kTwo], s[kTwo];
        turns.template at<Row::P, LPR>(q, m.b, m.t, l, c, s);
        // y_a = r (x_a ac - x_b bs), y_b = r (x_b bc + x_a as), from the weight of the heads that follow
        float2 ac[kTwo], as[kTwo], bc[kTwo], bs[kTwo];
        const auto weigh = [&](const float *w) {
            Row ws;
            if (w) ws.get(w, half, l);
            else ws.fill(1.0f);
#pragma unroll
            for (int i = 0; i < kTwo; i++) {
                bc[i] = mul2(c[i], ws.b[i]), bs[i] = neg2(mul2(s[i], ws.b[i]));
                ac[i] = mul2(c[i], ws.a[i]), as[i] = mul2(s[i], ws.a[i]);
            }
        };
        weigh(m.h0 < q.HQ ? q.wq : q.wk);
        const auto turn = [&](Row &v, float *to) {
            float r = 1.0f;
            if (q.norm) {
                float2 ss = mul2(v.a[0], v.a[0]);
                ss = fma2(v.b[0], v.b[0], ss);
#pragma unroll
                for (int i = 1; i < kTwo; i++) ss = fma2(v.b[i], v.b[i], fma2(v.a[i], v.a[i], ss));
                r = rsqrtf(fmaf(group_sum<LPR>(sum2(ss), lane, l), inv_d, q.eps));
            }
#pragma unroll
            for (int i = 0; i < kTwo; i++) {
                const float2 xa = mul2(v.a[i], both(r)), xb = mul2(v.b[i], both(r));
                v.a[i] = fma2(xa, ac[i], mul2(xb, bs[i]));
                v.b[i] = fma2(xb, bc[i], mul2(xa, as[i]));
            }
            if (m.live) v.put(to, half, l);
        };
        for (int h = m.h0;;) {
#pragma unroll
            for (int k = 0; k < U; k++) {
                if (h + k >= m.h1) break;
                if (h + k == q.HQ && h + k > m.h0) weigh(q.wk); // the key heads begin within the run
                turn(row[k], out + k * q.D);
            }
            h += U, x += U * q.sh, out += U * q.D;
            if (h >= m.h1) break;
#pragma unroll
            for (int k = 0; k < U; k++)
                if (h + k < m.h1) row[k].get(x + k * q.sh, half, l);
        }
    }
}

constexpr int kSumRows = 64; // rows whose terms of a weight's gradient a lane adds up in fp32

// part (may be NULL): the block's sums of g n over its query rows and over its key rows, [block][2][D]. A lane's fp32 sums
// go to sums of its own in 64 bits before an item could take them past kSumRows rows, so that the error does not grow
// with the number of rows (in fp32 alone it was 270 * 2^-24 of a sum of 80000 x 1000 rows, now below 92 for any number;
// both passes of 4 x 4680 x 24 heads of 128 take 190 us with it and 188 without).
template <int VEC, int LPR, bool INTER>
__global__ void __launch_bounds__(256, 2) k_rope_bwd(const __grid_constant__ nck_rope q, const RopeGrid g,
                                                  const float *dy, float *dx, int acc,
                                                  float *__restrict__ part) {
    constexpr int kPer = 32 / LPR, kGroups = 8 * kPer, U = VEC == 4 ? kRowsBwd : kRowsBwd - 1;
    typedef Own<VEC, LPR, INTER> Row;
    __shared__ double sums[4 * kOwn][256 + LPR]; // query heads' first elements of pairs, their second ones, key heads'
    const int lane = threadIdx.x & 31, l = lane % LPR, half = q.D >> 1;
    const float inv_d = 1.0f / (float)q.D;
    __shared__ Turns turns;
    turns.fill(q);
    cudaGridDependencySynchronize();
    Row sum[2]; // of query heads, of key heads
    sum[0].fill(0.0f), sum[1].fill(0.0f);
    int rows = 0; // added to them
    bool moved = false;
    const auto move = [&]() { // to 64 bits
#pragma unroll
        for (int side = 0; side < 2; side++) {
#pragma unroll
            for (int i = 0; i < kTwo; i++) {
                const float v[4] = {sum[side].a[i].x, sum[side].a[i].y, sum[side].b[i].x, sum[side].b[i].y};
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    double *to = &sums[(2 * side + (k >> 1)) * kOwn + 2 * i + (k & 1)][threadIdx.x];
                    *to = moved ? *to + (double)v[k] : (double)v[k];
                }
            }
            sum[side].fill(0.0f);
        }
        rows = 0, moved = true;
    };
    for (int64_t it = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); it < g.items; it += (int64_t)gridDim.x * 8) {
        const Item<LPR> m(q, g, it, lane / LPR);
        const float *x = q.x + m.b * q.sb + m.t * q.st + m.h0 * q.sh;
        const int64_t at = ((int64_t)m.tok * q.H + m.h0) * q.D;
        const float *from = dy + at;
        float *to = dx + at;
        Row x_row[U], dy_row[U]; // the first rows are on their way while the angles are formed
        const auto fetch = [&](int h) {
#pragma unroll
            for (int k = 0; k < U; k++)
                if (h + k < m.h1) x_row[k].get(x + k * q.sh, half, l), dy_row[k].get(from + k * q.D, half, l);
        };
        fetch(m.h0);
        float2 c[kTwo], s[kTwo];
        turns.template at<Row::P, LPR>(q, m.b, m.t, l, c, s);
        Row ws;
        const auto weigh = [&](const float *w) {
            if (w) ws.get(w, half, l);
            else ws.fill(1.0f);
        };
        weigh(m.h0 < q.HQ ? q.wq : q.wk);
        const auto turn_back = [&](Row &v, Row &d, float *to, Row &part_sum) {
            float2 ss = both(0.0f), dot = both(0.0f);
#pragma unroll
            for (int i = 0; i < kTwo; i++) {
                const float2 ya = d.a[i], yb = d.b[i];
                d.a[i] = fma2(ya, c[i], mul2(yb, s[i]));
                d.b[i] = fma2(yb, c[i], neg2(mul2(ya, s[i])));
                ss = fma2(v.a[i], v.a[i], fma2(v.b[i], v.b[i], ss));
                dot = fma2(mul2(d.a[i], ws.a[i]), v.a[i], fma2(mul2(d.b[i], ws.b[i]), v.b[i], dot));
            }
            float r = 1.0f, k = 0.0f; // dx = r g w + k x, k = -r^3 sum(g w x) / D
            if (q.norm) {
                const float all = group_sum<LPR>(sum2(ss), lane, l), mean = group_sum<LPR>(sum2(dot), lane, l) * inv_d;
                r = rsqrtf(fmaf(all, inv_d, q.eps));
                k = -(mean * r) * (r * r);
            }
            if (!m.live) return;
            Row o;
#pragma unroll
            for (int i = 0; i < kTwo; i++) {
                const float2 ga = mul2(d.a[i], both(r)), gb = mul2(d.b[i], both(r));
                part_sum.a[i] = fma2(ga, v.a[i], part_sum.a[i]);
                part_sum.b[i] = fma2(gb, v.b[i], part_sum.b[i]);
                o.a[i] = fma2(ga, ws.a[i], mul2(both(k), v.a[i]));
                o.b[i] = fma2(gb, ws.b[i], mul2(both(k), v.b[i]));
            }
            if (dx && acc) { // added to what is there
                v.get(to, half, l);
#pragma unroll
                for (int i = 0; i < kTwo; i++) {
                    o.a[i] = fma2(v.a[i], both(1.0f), o.a[i]);
                    o.b[i] = fma2(v.b[i], both(1.0f), o.b[i]);
                }
            }
            if (dx) o.put(to, half, l);
        };
        for (int h = m.h0;;) {
#pragma unroll
            for (int k = 0; k < U; k++) {
                if (h + k >= m.h1) break;
                if (h + k == q.HQ && h + k > m.h0) weigh(q.wk); // the key heads begin within the run
                if (h + k < q.HQ) turn_back(x_row[k], dy_row[k], to + k * q.D, sum[0]);
                else turn_back(x_row[k], dy_row[k], to + k * q.D, sum[1]);
            }
            h += U, x += U * q.sh, from += U * q.D, to += U * q.D;
            if (h >= m.h1) break;
            fetch(h);
        }
        if (part && (rows += g.run) > kSumRows - g.run) move();
    }
    if (!part) return;
    move();
    __syncthreads();
    // S neighbouring threads add up the groups' sums of one element
    constexpr int kAll = 4 * kOwn * LPR, S = kAll <= 16 ? 16 : kAll <= 32 ? 8 : kAll <= 64 ? 4 : kAll <= 128 ? 2 : 1;
    for (int at = threadIdx.x / S; at < (kAll + 255) / 256 * (256 / S); at += 256 / S) {
        const int k = at / LPR, lane_of = at % LPR, i = k % kOwn;
        double t = 0.0;
        if (at < kAll)
            for (int j = threadIdx.x % S; j < kGroups; j += S) t += sums[k][j / kPer * 32 + j % kPer * LPR + lane_of];
#pragma unroll
        for (int o = S / 2; o > 0; o >>= 1) t += __shfl_xor_sync(~0u, t, o);
        const int p = (i / Row::P * LPR + lane_of) * Row::P + i % Row::P; // the pair
        if (threadIdx.x % S || at >= kAll || p >= half) continue;
        const int side = k / (2 * kOwn), second = k / kOwn & 1;
        part[((int64_t)blockIdx.x * 2 + side) * q.D + (INTER ? 2 * p + second : p + second * half)] = (float)t;
    }
}

// dw (+)= the blocks' partial sums in a fixed order; 32 columns a block, 32 slices of the blocks each
__global__ void __launch_bounds__(1024) k_rope_dw(const float *part, int blocks, int D, float *dwq, int acc_q,
                                                  float *dwk, int acc_k) {
    __shared__ double red[32][33];
    cudaGridDependencySynchronize();
    const int lane = threadIdx.x & 31, sl = threadIdx.x >> 5, col = blockIdx.x * 32 + lane;
    double t = 0.0;
    if (col < 2 * D) {
        constexpr int U = 8; // loads in flight
        for (int b = sl; b < blocks; b += 32 * U) {
            float v[U];
#pragma unroll
            for (int u = 0; u < U; u++) v[u] = b + 32 * u < blocks ? part[(int64_t)(b + 32 * u) * 2 * D + col] : 0.0f;
#pragma unroll
            for (int u = 0; u < U; u++) t += (double)v[u];
        }
    }
    red[sl][lane] = t;
    __syncthreads();
    // warp sl sums column sl of the block
    t = red[lane][sl];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(~0u, t, o);
    const int c = blockIdx.x * 32 + sl;
    float *dw = c < D ? dwq : dwk;
    if (lane || c >= 2 * D || !dw) return;
    float *to = dw + (c < D ? c : c - D);
    const bool acc = c < D ? acc_q : acc_k;
    *to = acc ? *to + (float)t : (float)t;
}

bool aligned(const void *p, int vec) { return ((uintptr_t)p & (size_t)(4 * vec - 1)) == 0; }

// The widest vector that x's layout and every pointer of the pass allow: 4, 2 or 1 floats.
int vector_of(const nck_rope *q, const void *p1, const void *p2) {
    for (int vec = 4; vec > 1; vec >>= 1) {
        bool ok = q->D % (q->interleaved ? vec : 2 * vec) == 0 && aligned(q->x, vec) && aligned(q->wq, vec) && aligned(q->wk, vec) &&
                  aligned(p1, vec) && aligned(p2, vec);
        ok = ok && (q->B == 1 || q->sb % vec == 0) && (q->T == 1 || q->st % vec == 0) && (q->H == 1 || q->sh % vec == 0);
        if (ok) return vec;
    }
    return 1;
}

// All heads are one run when the tokens alone fill the GPU's resident warps, and even parts of them (down to single
// heads) when they do not: a shorter run forms the angles more often, a longer one leaves SMs idle.
// A pass that sums weight gradients has runs of at most `most` heads; two of them hold more than 64 heads' worth of the
// result, which is in memory, so there are fewer than 2^31 items.
RopeGrid split_of(const nck_dev *d, const nck_rope *q, int lpr, int most) {
    RopeGrid g;
    const int64_t tokens = q->B * q->T, per = 32 / lpr, tiles = (tokens + per - 1) / per;
    int64_t chunks = (int64_t)d->sm_count * 16 / tiles;
    chunks = chunks < 1 ? 1 : chunks > q->H ? q->H : chunks;
    g.run = (int)((q->H + chunks - 1) / chunks);
    if (g.run > most) g.run = most;
    g.tiles = (int)tiles;
    g.items = (q->H + g.run - 1) / g.run * tiles;
    g.by_tiles = make_fastdiv((uint32_t)tiles);
    g.by_T = make_fastdiv((uint32_t)q->T);
    return g;
}

template <int VEC, int LPR, bool INTER>
int launch(nck_dev *d, const nck_rope *q, float *y, const float *dy, float *dx, int acc, float *part) {
    static int room_fwd = 0, room_bwd = 0;
    if (!room_fwd) {
        room_bwd = resident_blocks(d, k_rope_bwd<VEC, LPR, INTER>, 256);
        room_fwd = resident_blocks(d, k_rope_fwd<VEC, LPR, INTER>, 256);
    }
    const RopeGrid g = split_of(d, q, LPR, part ? kSumRows : 65535);
    const int64_t blocks = (g.items + 7) / 8;
    const int room = y ? room_fwd : room_bwd, grid = (int)(blocks < room ? blocks : room);
    if (y) launch_early(d, k_rope_fwd<VEC, LPR, INTER>, grid, 256, *q, g, y);
    else launch_early(d, k_rope_bwd<VEC, LPR, INTER>, grid, 256, *q, g, dy, dx, acc, part);
    NCK_LAUNCHED(d, 1);
    return grid;
}

// As many lanes as a row needs at four pairs a lane, up to the number that lets as many rows share a warp.
template <int VEC, bool INTER>
int by_lanes(nck_dev *d, const nck_rope *q, float *y, const float *dy, float *dx, int acc, float *part) {
    switch (32 / ((q->D / 2 + kOwn - 1) / kOwn)) { // rows to a warp
    case 32: return launch<VEC, 1, INTER>(d, q, y, dy, dx, acc, part);
    case 16: return launch<VEC, 2, INTER>(d, q, y, dy, dx, acc, part);
    case 10: return launch<VEC, 3, INTER>(d, q, y, dy, dx, acc, part);
    case 8: return launch<VEC, 4, INTER>(d, q, y, dy, dx, acc, part);
    case 6: return launch<VEC, 5, INTER>(d, q, y, dy, dx, acc, part);
    case 5: return launch<VEC, 6, INTER>(d, q, y, dy, dx, acc, part);
    case 4: return launch<VEC, 8, INTER>(d, q, y, dy, dx, acc, part);
    case 3: return launch<VEC, 10, INTER>(d, q, y, dy, dx, acc, part);
    case 2: return launch<VEC, 16, INTER>(d, q, y, dy, dx, acc, part);
    default: return launch<VEC, 32, INTER>(d, q, y, dy, dx, acc, part);
    }
}

template <bool INTER>
int dispatch(nck_dev *d, const nck_rope *q, float *y, const float *dy, float *dx, int acc, float *part) {
    const int vec = y ? vector_of(q, y, nullptr) : vector_of(q, dy, dx);
    if (vec == 1) return by_lanes<1, INTER>(d, q, y, dy, dx, acc, part);
    if (vec == 2) return by_lanes<2, INTER>(d, q, y, dy, dx, acc, part);
    return by_lanes<4, INTER>(d, q, y, dy, dx, acc, part);
}

}  // namespace

extern "C" void nck_rope_fwd(nck_dev *d, const nck_rope *q, float *y) {
    const double n = (double)q->B * q->T * q->H * q->D;
    if (n == 0) return;
    Scope sc(d, "qk_norm_rope", 10.0 * n, 8.0 * n);
    if (q->interleaved) dispatch<true>(d, q, y, nullptr, nullptr, 0, nullptr);
    else dispatch<false>(d, q, y, nullptr, nullptr, 0, nullptr);
}

extern "C" void nck_rope_bwd(nck_dev *d, const nck_rope *q, const float *dy, float *dx, int acc_x, float *dwq, int acc_q,
                             float *dwk, int acc_k) {
    const double n = (double)q->B * q->T * q->H * q->D;
    Scope sc(d, "qk_norm_rope_bwd", 20.0 * n, 12.0 * n);
    float *part = dwq || dwk ? (float *)d->scratch : nullptr;
    int grid = 0;
    if (n > 0 && (dx || part))
        grid = q->interleaved ? dispatch<true>(d, q, nullptr, dy, dx, acc_x, part)
                              : dispatch<false>(d, q, nullptr, dy, dx, acc_x, part);
    if (!part) return;
    launch_early(d, k_rope_dw, (2 * q->D + 31) / 32, 1024, (const float *)part, grid, q->D, dwq, acc_q, dwk, acc_k);
    NCK_LAUNCHED(d, 1);
}
