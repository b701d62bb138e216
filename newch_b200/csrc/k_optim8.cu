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
// 28), so HBM bounds it as long as the arithmetic, about 100 instructions an element, keeps up. A warp owns a
// block: a lane holds eight elements as two float4 of w and g and two words of four codes each, the
// largest values are a warp's maximum, and nothing is read or written twice. The step itself is formed with the
// approximate division and root (each within 2 steps of fp32 of a term that is lr times w's size or less).
#include "k_common.cuh"

using namespace nck;

namespace {

constexpr int kBlock = NCK_OPT8_BLOCK;
constexpr float kUnitM = 1.0f / (127.0f * 127.0f), kUnitV = (float)(1.0 / (255.0 * 255.0 * 255.0 * 255.0));
constexpr float kFullM = 127.0f * 127.0f, kFullV = 255.0f * 255.0f * 255.0f * 255.0f;
constexpr float kLeast = 5.0487097934144756e-29f; // 2^-94: blocks whose largest value is below stand for zero
constexpr float kRound = 12582912.0f;             // 1.5 * 2^23: adding it rounds to whole numbers

__device__ __forceinline__ float root(float x) {
    float r;
    asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// byte k of a word of unsigned codes as a float
__device__ __forceinline__ float byte_of(uint32_t w, int k) {
    return __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7440u | (uint32_t)k)) - 8388608.0f;
}

// the low byte of a whole number |x| < 2^22
__device__ __forceinline__ uint32_t low_byte(float x) { return __float_as_uint(x + kRound); }

__device__ __forceinline__ uint32_t pack(const uint32_t (&b)[4]) {
    return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
}

__device__ __forceinline__ float decode_m(float s, float unit, float c) {
    const float v = unit * (c * fabsf(c));
    return fabsf(c) == 127.0f ? copysignf(s, c) : v;
}

__device__ __forceinline__ float decode_v(float s, float unit, float c) {
    const float q = c * c, v = (unit * q) * q;
    return c == 255.0f ? s : v;
}

// the code of |m| by its share (NaN gives some code of the range: its block's largest value is NaN as well)
__device__ __forceinline__ float code_m(float share) {
    float c = fminf(fmaxf(root(share), 0.0f), 127.0f);
    c = (c + kRound) - kRound;
    const float lo = c - 0.5f, hi = c + 0.5f;
    if (share < lo * lo && c > 0.0f) c -= 1.0f;
    if (share >= hi * hi && c < 127.0f) c += 1.0f;
    return c;
}

__device__ __forceinline__ float code_v(float share) {
    float c = fminf(fmaxf(root(root(share)), 0.0f), 255.0f);
    c = (c + kRound) - kRound;
    const float lo = c - 0.5f, hi = c + 0.5f, lo2 = lo * lo, hi2 = hi * hi;
    if (share < lo2 * lo2 && c > 0.0f) c -= 1.0f;
    if (share >= hi2 * hi2 && c < 255.0f) c += 1.0f;
    return c;
}

// The largest of non-negative values over a warp; NaN counts as larger than any.
__device__ __forceinline__ float warp_largest(const float (&v)[8]) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
    top = __reduce_max_sync(~0u, top);
    const float s = __uint_as_float(top);
    return s < kLeast ? 0.0f : s;
}

// Eight elements' moments to codes, and the block's largest values. m and v are the lane's elements (0 past the end).
__device__ __forceinline__ void encode(const float (&m)[8], const float (&v)[8], float &sm, float &sv, uint32_t (&cm)[2],
                                       uint32_t (&cv)[2]) {
    sm = warp_largest(m);
    sv = warp_largest(v);
    const float rm = sm > 0.0f ? (1.0f / sm) * kFullM : 0.0f, rv = sv > 0.0f ? (1.0f / sv) * kFullV : 0.0f;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        uint32_t bm[4], bv[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int i = 4 * h + k;
            const float c = code_m(fabsf(m[i]) * rm), d = code_v(v[i] * rv);
            bm[k] = low_byte(copysignf(c, m[i]));
            bv[k] = low_byte(v[i] > 0.0f && sv > 0.0f ? fmaxf(d, 1.0f) : 0.0f);
        }
        cm[h] = pack(bm);
        cv[h] = pack(bv);
    }
}

__device__ __forceinline__ void decode(uint32_t cm, uint32_t cv, float sm, float sv, float *m, float *v) {
    const float um = sm * kUnitM, uv = sv * kUnitV;
    cm ^= 0x80808080u; // signed bytes plus 128
#pragma unroll
    for (int k = 0; k < 4; k++) {
        m[k] = decode_m(sm, um, byte_of(cm, k) - 128.0f);
        v[k] = decode_v(sv, uv, byte_of(cv, k));
    }
}

__device__ __forceinline__ void get4(const float *p, int64_t n, int at, float (&v)[4]) {
    if (at + 4 <= n) {
        const float4 f = *reinterpret_cast<const float4 *>(p + at);
        v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = at + k < n ? p[at + k] : 0.0f;
    }
}

__device__ __forceinline__ void put4(float *p, int64_t n, int at, const float (&v)[4]) {
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

__global__ void __launch_bounds__(256) k_adamw8(Step8 h, nck_opt8 q, const nck_param_seg *__restrict__ segs,
                                                const nck_opt_chunk *__restrict__ chunks,
                                                const unsigned char *__restrict__ present) {
    const nck_opt_chunk c = chunks[blockIdx.x];
    const nck_param_seg s = segs[c.seg];
    if (present && !present[s.param]) return;
    const int lane = threadIdx.x & 31, off = (int)(threadIdx.x >> 5) * kBlock;
    if (off >= c.len) return;
    const int64_t blk = s.blk + (c.off + off) / kBlock;
    float *w = s.w + c.off + off;
    const float *g = s.g + c.off + off;
    const int64_t n = c.len - off < kBlock ? c.len - off : kBlock;
    uint32_t *pm = reinterpret_cast<uint32_t *>(q.cm + blk * kBlock), *pv = reinterpret_cast<uint32_t *>(q.cv + blk * kBlock);
    float wv[2][4], gv[2][4], m[8], v[8];
    uint32_t cm[2], cv[2];
    float sm = q.sm[blk], sv = q.sv[blk];
#pragma unroll
    for (int k = 0; k < 2; k++) {
        get4(w, n, k * 128 + lane * 4, wv[k]);
        get4(g, n, k * 128 + lane * 4, gv[k]);
        cm[k] = pm[k * 32 + lane];
        cv[k] = pv[k * 32 + lane];
    }
#pragma unroll
    for (int k = 0; k < 2; k++) {
        decode(cm[k], cv[k], sm, sv, m + 4 * k, v + 4 * k);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int j = 4 * k + i;
            const float gj = h.gs * gv[k][i];
            m[j] = h.beta1 * m[j] + h.up1 * gj;
            v[j] = h.beta2 * v[j] + h.up2 * gj * gj;
            const float step = __fdividef(h.rate * m[j], fmaf(root(v[j]), h.unbias2, h.eps));
            wv[k][i] = fmaf(wv[k][i], h.keep, -step);
        }
        put4(w, n, k * 128 + lane * 4, wv[k]);
    }
    encode(m, v, sm, sv, cm, cv);
#pragma unroll
    for (int k = 0; k < 2; k++) {
        pm[k * 32 + lane] = cm[k];
        pv[k * 32 + lane] = cv[k];
    }
    if (lane == 0) q.sm[blk] = sm, q.sv[blk] = sv;
}

// Codes to values (PUT false) or values to codes: m's at val[0], v's at val[second], a span's at its offset.
template <bool PUT>
__global__ void __launch_bounds__(256) k_opt8_values(nck_opt8 q, const nck_opt8_span *__restrict__ spans,
                                                     const nck_opt_chunk *__restrict__ chunks, float *val, int64_t second,
                                                     int dense) {
    const nck_opt_chunk c = chunks[blockIdx.x];
    const nck_opt8_span s = spans[c.seg];
    const int lane = threadIdx.x & 31, off = (int)(threadIdx.x >> 5) * kBlock;
    if (off >= c.len) return;
    const int64_t blk = s.blk + (c.off + off) / kBlock;
    float *pm_val = val + (dense ? s.dense : s.flat) + c.off + off, *pv_val = pm_val + second;
    const int n = c.len - off < kBlock ? c.len - off : kBlock;
    uint32_t *pm = reinterpret_cast<uint32_t *>(q.cm + blk * kBlock), *pv = reinterpret_cast<uint32_t *>(q.cv + blk * kBlock);
    float m[8], v[8];
    uint32_t cm[2], cv[2];
    if (PUT) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int at = (i >> 2) * 128 + lane * 4 + (i & 3);
            m[i] = at < n ? pm_val[at] : 0.0f;
            v[i] = at < n ? fabsf(pv_val[at]) : 0.0f;
        }
        float sm, sv;
        encode(m, v, sm, sv, cm, cv);
#pragma unroll
        for (int k = 0; k < 2; k++) pm[k * 32 + lane] = cm[k], pv[k * 32 + lane] = cv[k];
        if (lane == 0) q.sm[blk] = sm, q.sv[blk] = sv;
        return;
    }
    const float sm = q.sm[blk], sv = q.sv[blk];
#pragma unroll
    for (int k = 0; k < 2; k++) decode(pm[k * 32 + lane], pv[k * 32 + lane], sm, sv, m + 4 * k, v + 4 * k);
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int at = (i >> 2) * 128 + lane * 4 + (i & 3);
        if (at < n) pm_val[at] = m[i], pv_val[at] = v[i];
    }
}

}  // namespace

extern "C" void nck_adamw8_step(nck_dev *d, const nck_opt_hyper *h, const nck_opt8 *q, const nck_param_seg *dsegs,
                                const nck_opt_chunk *dchunks, int nchunk, int64_t total, const unsigned char *present) {
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
    k_adamw8<<<nchunk, 256, 0, NCK_STREAM(d)>>>(s, *q, dsegs, dchunks, present);
    NCK_LAUNCHED(d, 1);
}

extern "C" void nck_opt8_values(nck_dev *d, const nck_opt8 *q, const nck_opt8_span *dspans, const nck_opt_chunk *dchunks,
                                int nchunk, int64_t total, float *val, int64_t second, int dense, int put) {
    if (nchunk <= 0) return;
    Scope sc(d, put ? "opt8_put" : "opt8_get", 0.0, 10.0 * total);
    if (put) k_opt8_values<true><<<nchunk, 256, 0, NCK_STREAM(d)>>>(*q, dspans, dchunks, val, second, dense);
    else k_opt8_values<false><<<nchunk, 256, 0, NCK_STREAM(d)>>>(*q, dspans, dchunks, val, second, dense);
    NCK_LAUNCHED(d, 1);
}
