// AdamW with both moments in 8 bits: one launch for all parameters.
//
// A parameter is cut into blocks of 256 elements, the last one shorter. A block keeps the largest |m| and the
// largest v of its elements in fp32 and a byte for each element's share of them:
//   m = sign(c) s (c / 127)^2, c in [-127, 127];   v = s (c / 255)^4, c in [0, 255]
// The square spaces the steps of m by its size; the fourth power does the same for the root of v, which the
// update divides by: shares of sqrt(v) down to 1.5e-5 of the block's largest have codes, where even steps in v
// would end at 0.06 and even steps in sqrt(v) at 0.004. A v that is not zero never gets code 0: a rounded-off v
// would divide m by eps alone. A code is the number of borders (j - 1/2)^2, or (j - 1/2)^4, that the share times
// 127^2, or 255^4, reaches: borders are exact (or the rounded exact) fp32 numbers, and an approximate root only
// proposes a code that the two borders around it then settle, so the codes do not depend on how a root is
// computed. The share's products are written without fused multiply-adds; every code is a function of
// m, v, the gradient and the two largest values alone.
//
// The update reads w, g and two bytes and writes w and two bytes: 16 bytes an element (AdamW with fp32 moments:
// 28), so HBM bounds it as long as the arithmetic keeps up: at 6.5 TB/s an SM has about 90 issue slots for 32
// elements. A warp owns a block: a lane holds eight elements as two float4 of w and of g and the sixteen codes
// of them as one 16-byte word (the codes are stored in that order), the largest values are a warp's maximum, and
// nothing is read or written twice. A code's proposal is biased upward by 2^-20 of the root (the approximate
// root is off by 2^-22 at most), so one border settles it. Measured on 135M weights (2.16 GB a step): 360 us, 92% of
// the measured copy rate; with two-sided borders, denormal-safe roots and separate code arrays (116 issue slots an
// element) it was 560 us. The step itself is formed with the approximate division and root (each within 2 steps of
// fp32 of a term that is lr times w's size or less).
#include "k_common.cuh"

using namespace nck;

namespace {

constexpr int kBlock = NCK_OPT8_BLOCK;
constexpr float kUnitM = 1.0f / (127.0f * 127.0f), kUnitV = (float)(1.0 / (255.0 * 255.0 * 255.0 * 255.0));
constexpr float kFullM = 127.0f * 127.0f, kFullV = 255.0f * 255.0f * 255.0f * 255.0f;
constexpr float kLeast = 5.0487097934144756e-29f; // 2^-94: blocks whose largest value is below stand for zero
constexpr float kRound = 12582912.0f;             // 1.5 * 2^23: adding it rounds to whole numbers
constexpr float kUp = 1.0f + 9.5367431640625e-7f; // 1 + 2^-20

// off by 2^-23 of the root; arguments below 2^-126 have root 0
__device__ __forceinline__ float root(float x) {
    float r;
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

__device__ __forceinline__ float ratio(float a, float b) {
    float r;
    asm("div.approx.ftz.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// the larger of two, NaN when either is
__device__ __forceinline__ float larger(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// byte k of a word, less `zero`, as a float
__device__ __forceinline__ float byte_of(uint32_t w, int k, float zero) {
    return __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7440u | (uint32_t)k)) - (8388608.0f + zero);
}

// the low bytes of four words
__device__ __forceinline__ uint32_t pack(const float (&b)[4]) {
    return __byte_perm(__byte_perm(__float_as_uint(b[0]), __float_as_uint(b[1]), 0x0040),
                       __byte_perm(__float_as_uint(b[2]), __float_as_uint(b[3]), 0x0040), 0x5410);
}

// m's codes are stored plus 128
__device__ __forceinline__ float decode_m(uint32_t w, int k, float s, float unit) {
    const float c = byte_of(w, k, 128.0f), v = unit * (c * fabsf(c));
    return fabsf(c) == 127.0f ? copysignf(s, c) : v;
}

__device__ __forceinline__ float decode_v(uint32_t w, int k, float s, float unit) {
    const float c = byte_of(w, k, 0.0f), q = c * c, v = (unit * q) * q;
    return c == 255.0f ? s : v;
}

// A float whose low byte is the code of m, plus 128, by |m|'s share. (The border below code 0 is negative. A share of
// NaN gives some byte: its block's largest value is NaN as well.)
__device__ __forceinline__ float code_m(float m, float share) {
    const float t = fmaf(root(share), kUp, kRound), c = t - kRound, lo = c - 0.5f;
    const float settled = share < lo * fabsf(lo) ? c - 1.0f : c;
    return fmaf(settled, copysignf(1.0f, m), kRound + 128.0f);
}

// A float whose low byte is the code of v by its share, at least `least` when v is not zero.
__device__ __forceinline__ float code_v(float v, float share, float least) {
    const float t = fmaf(root(root(share)), kUp, kRound), lo = (t - kRound) - 0.5f, lo2 = lo * fabsf(lo);
    const float settled = share < lo2 * fabsf(lo2) ? t - 1.0f : t;
    return v > 0.0f ? fmaxf(settled, kRound + least) : settled;
}

// The largest of a warp's non-negative values; NaN counts as larger than any.
__device__ __forceinline__ float warp_largest(float top) {
    const float s = __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(top) & 0x7fffffffu));
    return s < kLeast ? 0.0f : s;
}

__device__ __forceinline__ float largest_of(const float (&v)[8]) {
    float a = fabsf(v[0]);
#pragma unroll
    for (int i = 1; i < 8; i++) a = larger(a, fabsf(v[i]));
    return warp_largest(a);
}

// The lane's eight elements' moments (0 past the end) to codes, and the block's largest values. `hold` is called, by
// all lanes, when the largest v is infinite, and may change v.
template <typename F>
__device__ __forceinline__ uint4 encode(const float (&m)[8], float (&v)[8], float2 &top, F hold) {
    top = make_float2(largest_of(m), largest_of(v));
    if (top.y == INFINITY) {
        hold();
        top.y = largest_of(v);
    }
    const float rm = top.x > 0.0f ? (1.0f / top.x) * kFullM : 0.0f, rv = top.y > 0.0f ? (1.0f / top.y) * kFullV : 0.0f;
    const float least = top.y > 0.0f ? 1.0f : 0.0f;
    uint32_t w[4];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        float bm[4], bv[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            bm[k] = code_m(m[4 * h + k], fabsf(m[4 * h + k]) * rm);
            bv[k] = code_v(v[4 * h + k], v[4 * h + k] * rv, least);
        }
        w[h] = pack(bm);
        w[2 + h] = pack(bv);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ void get4(const float *p, int n, int at, float *v) {
    if (at + 4 <= n) {
        const float4 f = *reinterpret_cast<const float4 *>(p + at);
        v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = at + k < n ? p[at + k] : 0.0f;
    }
}

__device__ __forceinline__ void put4(float *p, int n, int at, const float *v) {
    if (at + 4 <= n) {
        *reinterpret_cast<float4 *>(p + at) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (at + k < n) p[at + k] = v[k];
    }
}

struct Step8 {
    float gs, keep, beta1, up1, beta2, up2, rate, unbias2, eps;
};

__global__ void __launch_bounds__(256) k_adamw8(Step8 h, nck_opt8 q, const nck_opt8_chunk *chunks,
                                                const unsigned char *present) {
    cudaGridDependencySynchronize();
    const nck_opt8_chunk c = chunks[blockIdx.x];
    if (present && !present[c.param]) return;
    const int lane = threadIdx.x & 31, off = (int)(threadIdx.x >> 5) * kBlock, n = c.len - off;
    if (n <= 0) return;
    const int64_t blk = (int64_t)c.blk + (threadIdx.x >> 5);
    float *w = c.w + off;
    const float *g = c.g + off;
    uint4 *codes = reinterpret_cast<uint4 *>(q.codes + blk * 2 * kBlock) + lane;
    float2 *tops = reinterpret_cast<float2 *>(q.top) + blk;
    float wv[8], gv[8], m[8], v[8];
    float2 top = *tops;
    const uint4 old = *codes;
#pragma unroll
    for (int k = 0; k < 2; k++) {
        get4(g, n, k * 128 + lane * 4, gv + 4 * k);
        get4(w, n, k * 128 + lane * 4, wv + 4 * k);
    }
    const uint32_t words[4] = {old.x, old.y, old.z, old.w};
    const float um = top.x * kUnitM, uv = top.y * kUnitV;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float gj = h.gs * gv[i];
        m[i] = h.beta1 * decode_m(words[i >> 2], i & 3, top.x, um) + h.up1 * gj;
        v[i] = h.beta2 * decode_v(words[2 + (i >> 2)], i & 3, top.y, uv) + h.up2 * gj * gj;
        wv[i] = fmaf(wv[i], h.keep, -ratio(h.rate * m[i], fmaf(root(v[i]), h.unbias2, h.eps)));
    }
#pragma unroll
    for (int k = 0; k < 2; k++) put4(w, n, k * 128 + lane * 4, wv + 4 * k);
    // A finite gradient whose square is not (above about 6e20) would make its block's largest v infinite and the other
    // 255 elements' v with it: it is held as the largest float. (Asked of the largest alone: a test of every element
    // took 9 registers more.)
    const bool was_finite = top.y < INFINITY;
    *codes = encode(m, v, top, [&]() {
        if (!was_finite) return;
        float gj[8];
#pragma unroll
        for (int k = 0; k < 2; k++) get4(g, n, k * 128 + lane * 4, gj + 4 * k);
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (v[i] == INFINITY && fabsf(gj[i]) < INFINITY) v[i] = 3.402823466e38f;
    });
    if (lane == 0) *tops = top;
}

// The values of one moment of a block: float4 stores at 16-byte boundaries wherever `to` starts, so that a row of
// moments may begin at any element (135M weights' two moments 226 us, 1.35 GB; 240 with loads and stores in turn).
template <bool M>
__device__ __forceinline__ void emit(const uint32_t *codes, float *to, int n, float s, int lane) {
    const float unit = s * (M ? kUnitM : kUnitV);
    const uint32_t *mine = codes + (M ? 0 : 2);
    const auto group = [&](int g) { return mine[(g & 31) * 4 + (g >> 5)]; }; // codes of elements 4g .. 4g + 3
    const auto value = [&](uint32_t w, int k) { return M ? decode_m(w, k, s, unit) : decode_v(w, k, s, unit); };
    if (n < kBlock) {
        for (int e = lane; e < n; e += 32) {
            const uint32_t w = group(e >> 2) >> (8 * (e & 3));
            to[e] = value(w, 0);
        }
        return;
    }
    const int lead = (int)((16 - ((uintptr_t)to & 15)) & 15) >> 2; // elements before the first boundary
    uint32_t words[2]; // both on their way before anything is stored
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const int g = lane + 32 * k;
        words[k] = !lead ? group(g) : g < 63 ? __funnelshift_r(group(g), group(g + 1), 8 * lead) : 0;
    }
    const int e = lane < lead ? lane : kBlock - 4 + lane; // elements before the first and behind the last boundary
    const uint32_t end = lead && lane < 4 ? group(e >> 2) >> (8 * (e & 3)) : 0;
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const int g = lane + 32 * k;
        if (lead && g == 63) break;
        const uint32_t w = words[k];
        *reinterpret_cast<float4 *>(to + lead + 4 * g) = make_float4(value(w, 0), value(w, 1), value(w, 2), value(w, 3));
    }
    if (lead && lane < 4) to[e] = value(end, 0);
}

// Codes to values (PUT false) or values to codes: m's at val[0], v's at val[second], a span's at its offset.
template <bool PUT>
__global__ void __launch_bounds__(256) k_opt8_values(nck_opt8 q, const nck_opt8_span *spans,
                                                     const nck_opt_chunk *chunks, float *val, int64_t second,
                                                     int dense) {
    cudaGridDependencySynchronize();
    const nck_opt_chunk c = chunks[blockIdx.x];
    const nck_opt8_span s = spans[c.seg];
    const int lane = threadIdx.x & 31, off = (int)(threadIdx.x >> 5) * kBlock;
    const int n = c.len - off < kBlock ? c.len - off : kBlock;
    if (n <= 0) return;
    const int64_t blk = s.blk + (c.off + off) / kBlock;
    float *ms = val + (dense ? s.dense : s.flat) + c.off + off, *vs = ms + second;
    uint32_t *codes = reinterpret_cast<uint32_t *>(q.codes + blk * 2 * kBlock);
    float2 *tops = reinterpret_cast<float2 *>(q.top) + blk;
    if constexpr (PUT) {
        float m[8], v[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int at = (i >> 2) * 128 + lane * 4 + (i & 3);
            m[i] = at < n ? ms[at] : 0.0f;
            v[i] = at < n ? fabsf(vs[at]) : 0.0f;
        }
        float2 top;
        reinterpret_cast<uint4 *>(codes)[lane] = encode(m, v, top, []() {});
        if (lane == 0) *tops = top;
    } else {
        const float2 top = *tops;
        emit<true>(codes, ms, n, top.x, lane);
        emit<false>(codes, vs, n, top.y, lane);
    }
}

}  // namespace

extern "C" int nck_opt8_chunks(const nck_param_seg *segs, int nseg, nck_opt8_chunk *chunks) {
    int k = 0;
    for (int i = 0; i < nseg; i++)
        for (int64_t off = 0; off < segs[i].n; off += NCK_OPT8_CHUNK, k++) {
            if (!chunks) continue;
            const int64_t left = segs[i].n - off;
            chunks[k] = {segs[i].w + off, segs[i].g + off, (int32_t)(segs[i].blk + off / NCK_OPT8_BLOCK),
                         (int32_t)(left < NCK_OPT8_CHUNK ? left : NCK_OPT8_CHUNK), segs[i].param, 0};
        }
    return k;
}

extern "C" void nck_adamw8_step(nck_dev *d, const nck_opt_hyper *h, const nck_opt8 *q, const nck_opt8_chunk *dchunks,
                                int nchunk, int64_t total, const unsigned char *present) {
    if (nchunk <= 0) return;
    Scope sc(d, "adamw8", 0.0, 16.0 * total);
    Step8 s;
    s.gs = h->gs;
    s.keep = 1.0f - h->lr * h->weight_decay;
    s.beta1 = h->beta1, s.up1 = 1.0f - h->beta1;
    s.beta2 = h->beta2, s.up2 = 1.0f - h->beta2;
    s.rate = h->lr / h->bc1;
    s.unbias2 = 1.0f / sqrtf(h->bc2);
    s.eps = h->eps;
    launch_early(d, k_adamw8, nchunk, 256, s, *q, dchunks, present);
    NCK_LAUNCHED(d, 1);
}

extern "C" void nck_opt8_values(nck_dev *d, const nck_opt8 *q, const nck_opt8_span *dspans, const nck_opt_chunk *dchunks,
                                int nchunk, int64_t total, float *val, int64_t second, int dense, int put) {
    if (nchunk <= 0) return;
    Scope sc(d, put ? "opt8_put" : "opt8_get", 0.0, 10.0 * total);
    if (put) launch_early(d, k_opt8_values<true>, nchunk, 256, *q, dspans, dchunks, val, second, dense);
    else launch_early(d, k_opt8_values<false>, nchunk, 256, *q, dspans, dchunks, val, second, dense);
    NCK_LAUNCHED(d, 1);
}
