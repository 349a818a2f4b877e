// kv8.hip - the 8-bit K/V cache: store, load, and the attention that reads it.
// Launchers are declared in kernels.h; their host checks are in hip.c.
//
// Layout (surge.h): records of 16 positions x one kv head, 16 hd key codes
// then 16 hd value codes, each in the order in which a wave's lanes take them
// as a matrix operand: 1 KB runs of 16 bytes per lane, so every fragment is
// one coalesced load and needs no shuffle.
//   keys    [hd/64][lane group 4][position 16][dim 16]: the A operand of
//           v_mfma_i32_16x16x64_i8 (lane (li, lg): row li, bytes 16 lg ..);
//   values  [hd/64][lane group 4][dim 16][dim tile 4][position 4]: dword j of
//           lane (li, lg) holds dim 16 j + li of positions 4 lg .. 4 lg + 3,
//           the positions whose scores that lane gets from the score product.
#include "devutil.h"
#include "kernels.h"

#define KV8_T SGK_KV8_TILE

__device__ __forceinline__ size_t rec_at(uint32_t tile, uint32_t n_kv, uint32_t h, uint32_t hd) {
    return ((size_t)tile * n_kv + h) * (2 * KV8_T) * hd;
}
__device__ __forceinline__ uint32_t key_at(uint32_t r, uint32_t d) {
    return (d / 64) * 1024 + (d / 16 % 4) * 256 + r * 16 + d % 16;
}
__device__ __forceinline__ uint32_t val_at(uint32_t r, uint32_t d) {
    return (d / 64) * 1024 + (r / 4) * 256 + (d % 16) * 16 + (d / 16 % 4) * 4 + r % 4;
}

// What a launch is divided by, with floor(2^32 / d) + 1 (2^32 / d where that is
// whole): the compiler's division of any two numbers is some 25 dependent
// instructions, and a wave has several before its first load.
struct kv8_div { uint32_t d, inv; };
__device__ __forceinline__ uint32_t div_by(uint32_t n, kv8_div v) {     // n < 2^31
    const uint32_t q = v.d == 1 ? n : __umulhi(n, v.inv);
    return q - (q * v.d > n);
}
static kv8_div kv8_div_of(uint32_t d) { return (kv8_div){d, d > 1 ? UINT32_MAX / d + 1 : 0}; }

// ---------------------------------------------------------------------------
// Store. One workgroup per (block, kv head, half) holds the block's new rows
// in registers: one read for the maximum and the codes. Keys go four dims of a
// row at a time, a wave taking 8 rows x 32 dims (whole lines of the rows, 128
// bytes of codes at a time); values 4 positions x 4 dims, transposed in
// registers into a dword per dim. 4 U fours per thread. Rows before base keep
// their codes unless the scale grows. Bound by memory: 8190 rows of 4 x 256 (84
// MB) 24.5 us in a trace with fresh inputs, 18 with the rows in the last cache;
// a copy of as many bytes takes 17-18. One row 4.2: load, maximum, codes in turn.
// ---------------------------------------------------------------------------
struct kv8_store_args {
    const float *x[2];
    int8_t *codes;
    float *scales;
    uint64_t stride;
    uint32_t n_kv, hd, block, base, n, hs, bs;      // hs, bs: log2 of hd and block
    kv8_div kv;
};

// Where four of a wave's keys lie: chunk c is 8 rows x 32 dims.
__device__ __forceinline__ void key_four(uint32_t c, uint32_t hs, uint32_t &r, uint32_t &d) {
    const uint32_t lane = threadIdx.x & 63;
    r = (c >> (hs - 5)) * 8 + lane / 8;
    d = (c & ((1u << (hs - 5)) - 1)) * 32 + lane % 8 * 4;
}

// Four x / s to the nearest integers, ties to even, as bytes. q = rint(x * (1/s))
// can be wrong only where x / s is within 2^-16 of a tie; there the remainder
// x - q s, exact in one fma, decides.
__device__ __forceinline__ uint32_t quant4(f32x4 x, float s, float inv) {
    float q[4], far = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const float t = x[e] * inv;
        q[e] = rintf(t);
        far = fmaxf(far, fabsf(t - q[e]));
    }
    if (!(far < 0.4999f)) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float r = fmaf(-q[e], s, x[e]), a = 2.0f * fabsf(r);
            if (a > s || (a == s && ((int)q[e] & 1))) q[e] += copysignf(1.0f, r);
        }
    }
    const uint32_t lo = __builtin_amdgcn_perm((uint32_t)(int)q[1], (uint32_t)(int)q[0], 0x0C0C0400u);
    const uint32_t hi = __builtin_amdgcn_perm((uint32_t)(int)q[3], (uint32_t)(int)q[2], 0x0C0C0400u);
    return lo | hi << 16;
}
__device__ __forceinline__ uint32_t requant4(uint32_t c, double was, double s) {
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) w |= (uint32_t)((int)rint((double)(int8_t)(c >> (8 * e)) * was / s) & 0xFF) << (8 * e);
    return w;
}
// bytes of a where the mask's bytes are set, else of b
__device__ __forceinline__ uint32_t pick_bytes(uint32_t mask, uint32_t a, uint32_t b) { return (a & mask) | (b & ~mask); }

// Workgroups in the order of the rows in memory: a block's heads and halves side by side.
// NTH threads, 4 U fours each: a large block takes more threads, not more
// registers (8190 rows of 4 heads of 256 in blocks of 64: 25 us with 4 units in
// each of 256 threads, 140 registers). With one unit six waves fit a SIMD (8 x
// 128, blocks of 16 27.9 -> 26.4 us a call); with two they would spill.
template <int U, int NTH>
__global__ void __launch_bounds__(NTH, U == 1 ? 6 : 4) k_kv8_store(kv8_store_args a, uint32_t first, int al) {
    __shared__ uint32_t red[NTH / 64];
    const uint32_t id = first + blockIdx.x, t = threadIdx.x, half = id & 1, hd = a.hd, unit = div_by(id / 2, a.kv), h = id / 2 - unit * a.n_kv;
    const uint32_t blk = (a.base >> a.bs) + unit, p0 = blk << a.bs;
    const uint32_t lo = max(p0, a.base), hi = (uint32_t)min((uint64_t)p0 + a.block, (uint64_t)a.base + a.n);
    const uint32_t kept = lo - p0, rows = hi - p0;      // rows kept .. rows-1 of the block are new
    const uint32_t fours = hd << a.bs >> 2, ds = a.hs - 2, dm = hd / 4 - 1;
    const float *x = a.x[half] + (size_t)(lo - a.base) * a.stride + (size_t)h * hd;
    float *sp = a.scales + ((size_t)blk * a.n_kv + h) * 2 + half;
    const float was = kept ? *sp : 0.0f;
    int8_t *codes = a.codes + (size_t)half * KV8_T * hd;
    f32x4 v[4 * U];
    uint32_t old[U][4], mx = 0;
#pragma unroll
    for (int i = 0; i < 4 * U; i++) {
        uint32_t r, d;
        const bool in = half ? (t + i / 4 * NTH) * 4 < fours : (t + i * NTH) < fours;
        if (half) { r = ((t + i / 4 * NTH) >> ds) * 4 + i % 4; d = ((t + i / 4 * NTH) & dm) * 4; }
        else key_four((t >> 6) + i * (NTH / 64), a.hs, r, d);
        v[i] = (f32x4){0.f, 0.f, 0.f, 0.f};
        if (in && r >= kept && r < rows) v[i] = ld4(x + (size_t)(r - kept) * a.stride + d, al);
    }
    // the dwords of values that hold rows which are not new, asked for early
    auto load_old = [&](int u, uint32_t r, uint32_t d) {
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (r < rows && (r < kept || r + 4 > rows))
                old[u][e] = *(const uint32_t *)(codes + rec_at((p0 + r) / KV8_T, a.n_kv, h, hd) + val_at(r % KV8_T, d + e));
    };
    if (half && (kept || rows < a.block)) {
#pragma unroll
        for (int u = 0; u < U; u++) load_old(u, ((t + u * NTH) >> ds) * 4, ((t + u * NTH) & dm) * 4);
    }
#pragma unroll
    for (int i = 0; i < 4 * U; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) mx = max(mx, __float_as_uint(v[i][e]) & 0x7FFFFFFFu);
    mx = wave_umax(mx);
    if ((t & 63) == 0) red[t >> 6] = mx;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NTH / 64; w++) mx = max(mx, red[w]);
    // 65520 and above round to infinity in f16; NaN's bits are above those
    const bool poison = mx >= 0x477FF000u || was != was;
    const float s = fmaxf(__uint_as_float(poison ? 0 : mx) * (1.0f / 127.0f), poison ? 0.0f : was);
    const bool grew = kept && s > was && !poison;
    if (t == 0) *sp = poison ? NAN : s;
    // a scale near the end of the range: x / s is the same for both times 2^64
    const float up = s < 0x1p-60f ? 0x1p64f : 1.0f, sq = s * up, inv = s > 0.0f ? 1.0f / sq : 0.0f;
    const bool zero = poison || s == 0.0f;
    const float sz = zero ? 1.0f : sq;
    if (zero || up != 1.0f) {
        const float top = zero ? 0.0f : 127.0f * sz;    // there the scale's own rounding may leave |x / s| above 127
#pragma unroll
        for (int i = 0; i < 4 * U; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) v[i][e] = __builtin_amdgcn_fmed3f(v[i][e] * up, -top, top);
    }
    if (!half) {
#pragma unroll
        for (int i = 0; i < 4 * U; i++) {
            uint32_t r, d;
            key_four((t >> 6) + i * (NTH / 64), a.hs, r, d);
            if (t + i * NTH >= fours || r >= rows || (r < kept && !grew)) continue;
            uint32_t *p = (uint32_t *)(codes + rec_at((p0 + r) / KV8_T, a.n_kv, h, hd) + key_at(r % KV8_T, d));
            *p = r < kept ? requant4(*p, was, s) : quant4(v[i], sz, inv);
        }
        return;
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const uint32_t r = ((t + u * NTH) >> ds) * 4, d = ((t + u * NTH) & dm) * 4;
        if ((t + u * NTH) * 4 >= fours || r >= rows || (r + 4 <= kept && !grew)) continue;
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; j++) w[j] = quant4(v[4 * u + j], sz, inv);
        // rows to dims: a 4 x 4 transpose of bytes
        const uint32_t a01 = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u), a23 = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u);
        const uint32_t b01 = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u), b23 = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
        uint32_t c[4] = {__builtin_amdgcn_perm(a23, a01, 0x05040100u), __builtin_amdgcn_perm(a23, a01, 0x07060302u),
                         __builtin_amdgcn_perm(b23, b01, 0x05040100u), __builtin_amdgcn_perm(b23, b01, 0x07060302u)};
        if (r < kept || r + 4 > rows) {     // some of the four rows are not new
            uint32_t isnew = 0, iskept = 0;
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) {
                if (r + j >= kept && r + j < rows) isnew |= 0xFFu << (8 * j);
                if (r + j < kept) iskept |= 0xFFu << (8 * j);
            }
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint32_t o = old[u][e], k = grew && iskept ? pick_bytes(iskept, requant4(o, was, s), o) : o;
                c[e] = pick_bytes(isnew, c[e], k);
            }
        }
#pragma unroll
        for (int e = 0; e < 4; e++)
            *(uint32_t *)(codes + rec_at((p0 + r) / KV8_T, a.n_kv, h, hd) + val_at(r % KV8_T, d + e)) = c[e];
    }
}

extern "C" hipError_t sgk_kv8_store(const float *k, const float *v, uint64_t stride, int8_t *codes, float *scales,
                                    uint32_t n_kv, uint32_t hd, uint32_t block, uint32_t base, uint32_t n, hipStream_t s,
                                    hipEvent_t done) {
    if (!n) return hipSuccess;
    if (!sgk_kv8_shape_ok(n_kv, hd, block) || ((uintptr_t)codes & 15)) return hipErrorInvalidValue;
    kv8_store_args a = {{k, v}, codes, scales, stride, n_kv, hd, block, base, n, (uint32_t)__builtin_ctz(hd), (uint32_t)__builtin_ctz(block), kv8_div_of(n_kv)};
    const int al = !((uintptr_t)k & 15) && !((uintptr_t)v & 15) && stride % 4 == 0;
    const uint64_t wgs = (((uint64_t)base + n + block - 1) / block - base / block) * n_kv * 2;
    if (wgs > UINT32_MAX) return hipErrorInvalidValue;
    const uint32_t units = block * hd / 16;
    for (uint64_t first = 0; first < wgs; first += 1u << 21) {      // a launch has fewer than 2^32 threads
        const dim3 grid((uint32_t)(wgs - first < 1u << 21 ? wgs - first : 1u << 21));
        const hipEvent_t ev = first + (1u << 21) < wgs ? NULL : done;
#define SC(U, N) launch(k_kv8_store<U, N>, grid, N, s, ev, a, (uint32_t)first, al)
        if (units <= 256) SC(1, 256);
        else if (units <= 512) SC(2, 256);
        else if (units <= 1024) SC(2, 512);
        else SC(2, 1024);
#undef SC
    }
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Load: hd threads per (tile, kv head, half), whole waves; fours as above. Bound
// by memory: the 84 MB above 15.1 us, 5.6 TB/s; one block 3.0.
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(TPB) k_kv8_load(const int8_t *codes, const float *scales, float *k, float *v,
                                                  uint64_t stride, kv8_div kv, uint32_t hd, uint32_t block,
                                                  uint32_t base, uint32_t n, uint32_t first, uint32_t halves, int al) {
    const uint32_t hs = __builtin_ctz(hd), id = first + ((blockIdx.x * TPB + threadIdx.x) >> hs);
    if (id >= halves) return;
    const uint32_t i = threadIdx.x & (hd - 1), half = id & 1, rec = id / 2;
    const uint32_t n_kv = kv.d, unit = div_by(rec, kv), tile = base / KV8_T + unit, h = rec - unit * n_kv;
    const float s = scales[((size_t)(tile >> __builtin_ctz(block / KV8_T)) * n_kv + h) * 2 + half];
    const int8_t *c = codes + rec_at(tile, n_kv, h, hd) + (size_t)half * KV8_T * hd;
    float *out = (half ? v : k) + (size_t)h * hd;
    const uint64_t p0 = (uint64_t)tile * KV8_T, end = (uint64_t)base + n;
    uint32_t w[4], r[4], d[4];
    if (!half) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            key_four((i >> 6) + j * (hd / 64), hs, r[j], d[j]);
            w[j] = *(const uint32_t *)(c + key_at(r[j], d[j]));
        }
    } else {
        const uint32_t r0 = (i >> (hs - 2)) * 4, d0 = (i & (hd / 4 - 1)) * 4;
        uint32_t b[4];
#pragma unroll
        for (int e = 0; e < 4; e++) b[e] = *(const uint32_t *)(c + val_at(r0, d0 + e));
        const uint32_t a01 = __builtin_amdgcn_perm(b[1], b[0], 0x05010400u), a23 = __builtin_amdgcn_perm(b[3], b[2], 0x05010400u);
        const uint32_t b01 = __builtin_amdgcn_perm(b[1], b[0], 0x07030602u), b23 = __builtin_amdgcn_perm(b[3], b[2], 0x07030602u);
        w[0] = __builtin_amdgcn_perm(a23, a01, 0x05040100u);
        w[1] = __builtin_amdgcn_perm(a23, a01, 0x07060302u);
        w[2] = __builtin_amdgcn_perm(b23, b01, 0x05040100u);
        w[3] = __builtin_amdgcn_perm(b23, b01, 0x07060302u);
#pragma unroll
        for (int j = 0; j < 4; j++) { r[j] = r0 + j; d[j] = d0; }
    }
#pragma unroll
    for (int j = 0; j < 4; j++) {
        if (p0 + r[j] < base || p0 + r[j] >= end) continue;
        st4(out + (size_t)(p0 + r[j] - base) * stride + d[j],
            (f32x4){(int8_t)w[j] * s, (int8_t)(w[j] >> 8) * s, (int8_t)(w[j] >> 16) * s, (int8_t)(w[j] >> 24) * s}, al);
    }
}

extern "C" hipError_t sgk_kv8_load(const int8_t *codes, const float *scales, float *k, float *v, uint64_t stride,
                                   uint32_t n_kv, uint32_t hd, uint32_t block, uint32_t base, uint32_t n, hipStream_t s,
                                   hipEvent_t done) {
    if (!n) return hipSuccess;
    if (!sgk_kv8_shape_ok(n_kv, hd, block) || ((uintptr_t)codes & 15)) return hipErrorInvalidValue;
    const int al = !((uintptr_t)k & 15) && !((uintptr_t)v & 15) && stride % 4 == 0;
    const uint32_t tiles = (uint32_t)(((uint64_t)base + n + KV8_T - 1) / KV8_T) - base / KV8_T;
    const uint64_t halves = (uint64_t)tiles * n_kv * 2;
    const uint32_t most = 1u << 20;         // of a launch: fewer than 2^32 threads
    if (halves > UINT32_MAX - most) return hipErrorInvalidValue;
    for (uint64_t first = 0; first < halves; first += most) {
        const uint64_t m = halves - first < most ? halves - first : most;
        launch(k_kv8_load, dim3((uint32_t)((m * hd + TPB - 1) / TPB)), TPB, s, first + most < halves ? NULL : done, codes, scales, k, v,
               stride, kv8_div_of(n_kv), hd, block, base, n, (uint32_t)first, (uint32_t)(first + m), al);
    }
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Attention of few rows: decode, and small chunks. A workgroup takes 16 rows
// (token-major, the query heads of one kv head inside a token) and a part of
// the keys. Every wave streams its own steps of 32 keys straight from the
// cache into operands:
//  - q in fixed point against its row's largest element, 24 bits as three int8
//    digits (q = sq (65536 d2 + 256 d1 + d0)): the score product is three
//    v_mfma_i32_16x16x64_i8 on the key codes as they lie, its sums exact, and
//    the keys are never converted;
//  - S^T = K Q^T leaves lane (li, lg) row li's scores of keys 4 lg .. 4 lg + 3
//    of both tiles, the order of the value records' dwords, so V^T P^T runs on
//    v_mfma_f32_16x16x32_f16 with the codes as f16 (exact) and p in two halves;
//  - the values' scale s_V = g 2^e goes into the weights: w = 2^(score + e - m)
//    g 2^13 with m an integer near the maximum of score + e, renewed where a
//    weight would pass 2^15.5. So w is in f16's range whatever the scales are,
//    while the sum of the softmax's own weights, w / s_V, at most 2^95 a key (e >=
//    -79), stays in f32's. e - m and the rescaling by 2^(m - m') are exact, and no
//    rounding is common to a block's keys; those of the exponents, half a step of
//    score + e - m each, are small where a weight is large. 2^13 keeps w's lower
//    half above f16's subnormals down to 2^-25 of the largest.
// No barrier or LDS in the key loop; the waves' maxima, sums and outputs join
// at the end. Bound by the cache's bytes: 262000 keys of 4 x 256 (537 MB) 85 us,
// 6.3 TB/s, where a plain read reaches 6.6; 32771 of 8 x 128 (67 MB) 14.1, with
// the waves' start and end in it; 700 of 2 x 256 6.0, one step's chain: 2 us to
// the loads' arrival, then 0.4 in the softmax, 0.7 in either product, 0.9 to join.
// ---------------------------------------------------------------------------
struct kv8_part {
    float *m, *s, *acc;         // [token][head][split] maxima and sums, [..][hd] outputs; NULL: one split
    kv8_div group, splits;      // query heads of a kv head
};
// Part sp of n units: the first n % splits parts have one more.
__device__ __forceinline__ void part_of(uint32_t n, uint32_t sp, kv8_div splits, uint32_t &first, uint32_t &end) {
    const uint32_t q = div_by(n, splits), more = n - q * splits.d;
    first = sp * q + min(sp, more);
    end = first + q + (sp < more);
}

#define KV8_P2 13
#define KV8_OVER 2.5f       // how far an exponent may pass the maximum kept before that is renewed: weights below 2^15.5
// A block's scale of values as its keys' weights take it.
struct v_scale { float e, g, rs; };         // exponent, 2^KV8_P2 mantissa, 2^KV8_P2 / 2^e
__device__ __forceinline__ v_scale v_scale_of(float s) {
    float a;
    asm("v_max_f32 %0, |%1|, %2" : "=v"(a) : "v"(s), "s"(0x1p-80f));          // zero as if tiny
    const int e = __builtin_amdgcn_frexp_expf(a);
    return (v_scale){(float)e, __builtin_amdgcn_ldexpf(s, KV8_P2 - e), __builtin_amdgcn_ldexpf(1.0f, KV8_P2 - e)};     // NaN stays in g
}

// 16 f32 of a row as the three digits' operand bytes: with 0x808080 added, the
// bytes of round(x inv) are its balanced digits plus 128, carries and all.
__device__ __forceinline__ void q_digits(const float (&x)[16], float inv, v4i &d0, v4i &d1, v4i &d2) {
#pragma unroll
    for (int w = 0; w < 4; w++) {
        uint32_t t[4];
#pragma unroll
        for (int e = 0; e < 4; e++) t[e] = (uint32_t)rintf(fmaf(x[4 * w + e], inv, 8421504.0f));    // 0x808080
        // bytes 0 and 1 of two elements, then byte 2; perm picks 0-3 from its second argument, 4-7 from its first
        const uint32_t a = __builtin_amdgcn_perm(t[1], t[0], 0x05010400u), b = __builtin_amdgcn_perm(t[3], t[2], 0x05010400u);
        const uint32_t c = __builtin_amdgcn_perm(t[1], t[0], 0x0C0C0602u), d = __builtin_amdgcn_perm(t[3], t[2], 0x0C0C0602u);
        d0[w] = (int)(__builtin_amdgcn_perm(b, a, 0x05040100u) ^ 0x80808080u);
        d1[w] = (int)(__builtin_amdgcn_perm(b, a, 0x07060302u) ^ 0x80808080u);
        d2[w] = (int)(__builtin_amdgcn_perm(d, c, 0x05040100u) ^ 0x80808080u);
    }
}
// The largest magnitude of three, NaN if one is.
__device__ __forceinline__ float amax3(float a, float b, float c) {
    float r;
    asm("v_maximum3_f32 %0, |%1|, |%2|, |%3|" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
// A row's q, spread over the four lanes of its column. Asked for before the
// first keys and values, which would otherwise have to arrive first.
template <int NC>
__device__ __forceinline__ void q_load(const float *q, bool al, uint32_t lg, float (&x)[NC][16]) {
    q += 16 * lg;
    if (al) {
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const f32x4 v = *(const f32x4 *)(q + 64 * c + 4 * w);
#pragma unroll
                for (int e = 0; e < 4; e++) x[c][4 * w + e] = v[e];
            }
    } else {
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int e = 0; e < 16; e++) x[c][e] = q[64 * c + e];
    }
}
// It as digits; returns the factor of the integer scores, sq * |mul|, NaN if an
// element is not finite.
#define KV8_QMAX (127.0f * 65536.0f)        // the row's largest element in units of its digits
template <int NC>
__device__ __forceinline__ float q_row(float (&x)[NC][16], float mul, v4i (&d)[3][NC]) {
    float mx[NC];
#pragma unroll
    for (int c = 0; c < NC; c++) {
        mx[c] = 0.0f;
#pragma unroll
        for (int e = 0; e < 16; e += 2) mx[c] = amax3(x[c][e], x[c][e + 1], mx[c]);
    }
    float am = mx[0];
#pragma unroll
    for (int c = 1; c < NC; c++) am = amax3(am, mx[c], 0.0f);
    am = amax3(am, swap16f(am), 0.0f);
    am = amax3(am, swap32f(am), 0.0f);
    const bool bad = !(am < INFINITY);
    if (bad) am = 0.0f;
    float up = 1.0f;
    if (__builtin_amdgcn_ballot_w64(am < 0x1p-60f)) {   // a row near the end of the range, times 2^64
        up = am < 0x1p-60f ? 0x1p64f : 1.0f;
        am *= up;
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int e = 0; e < 16; e++) x[c][e] *= up;
    }
    const float inv = am > 0.0f ? copysignf(KV8_QMAX / am, mul) : 0.0f;       // a negative scale turns q
#pragma unroll
    for (int c = 0; c < NC; c++) q_digits(x[c], inv, d[0][c], d[1][c], d[2][c]);
    return bad ? NAN : am / KV8_QMAX * fabsf(mul) / up;
}
// The score sums of the three digits as one float. The lowest's starts at the bits
// of 1.5 2^23, so that it comes out as a float, that much larger (it is
// below 2^22, 128 x 127 x 256); the highest's starts at that much less, in its
// units: a conversion a score less (a2 * 256 + a1 < 2^31).
struct q_start { v4i lo, hi; };
__device__ __forceinline__ q_start q_starts() {
    q_start s = {{0x4B400000, 0x4B400000, 0x4B400000, 0x4B400000}, {-192, -192, -192, -192}};
    asm volatile("" : "+v"(s.lo), "+v"(s.hi));      // in registers, not made again for every sum
    return s;
}
__device__ __forceinline__ float q_join(int a0, int a1, int a2) { return fmaf((float)(a2 * 256 + a1), 256.0f, __int_as_float(a0)); }
// eight codes (two dwords) as f16: the byte + 128 under 1024's exponent, less 1152
__device__ __forceinline__ f16x8 codes_f16(uint32_t a, uint32_t b) {
    const f16x2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
    const uint32_t ua = a ^ 0x80808080u, ub = b ^ 0x80808080u;
    f16x8 r;
    auto put = [&](int at, uint32_t u, uint32_t sel) {
        const f16x2 v = __builtin_bit_cast(f16x2, (uint32_t)__builtin_amdgcn_perm(0x64646464u, u, sel)) - off;
        r[at] = v[0];
        r[at + 1] = v[1];
    };
    put(0, ua, 0x04010400u);
    put(2, ua, 0x04030402u);
    put(4, ub, 0x04010400u);
    put(6, ub, 0x04030402u);
    return r;
}

// Exponents up to 2^20 are exact enough next to each other. Past that a maximum m
// may be rounded by more than the scale's exponent, e, so far rows have their
// weights times 2^-8 (2^-KV8_OFF), in which the usual scales' e fits.
#define KV8_FAR 0x1p20f
#define KV8_OFF 8.0f
__device__ __forceinline__ float far_off(float m) { return fabsf(m) > KV8_FAR && m != -INFINITY ? KV8_OFF : 0.0f; }
// The largest scale of keys with which no row of a wave can be far.
__device__ __forceinline__ float ks_most(float qf, uint32_t hd) {
    float m = qf;
    m = fmaxf(m, __uint_as_float(dppu<0xB1>(__float_as_uint(m))));
    m = fmaxf(m, __uint_as_float(dppu<0x4E>(__float_as_uint(m))));
    m = fmaxf(m, __uint_as_float(dppu<0x141>(__float_as_uint(m))));
    m = fmaxf(m, __uint_as_float(dppu<0x128>(__float_as_uint(m))));
    return fminf(KV8_FAR / (KV8_QMAX * 127.0f) / (float)hd * __builtin_amdgcn_rcpf(m), 0x1.fffffep127f);
}
// Whether a record's scales, by their bits, are those of the usual case: keys'
// zero or positive and no larger than that, values' finite and at least 2^-80;
// and the values' of that case, in scalar registers.
__device__ __forceinline__ bool scales_usual(uint32_t ks, uint32_t vs, uint32_t most) {
    return ks <= most && vs - 0x17800000u <= 0x7F7FFFFFu - 0x17800000u;
}
__device__ __forceinline__ v_scale v_scale_usual(uint32_t s) {
    const uint32_t e = s >> 23;
    return (v_scale){(float)((int)e - 126), __uint_as_float((s & 0x7FFFFFu) | (126u + KV8_P2) << 23), __uint_as_float((253u + KV8_P2 - e) << 23)};
}

// p g as f16 and what is left of it, four of a row: elements at .. at + 3 of the
// operands, together to 2^-22 of p g. (A mixed fma for the first half would take
// two products' and the conversion's cycles, 8.3 against 2.4 and 4.4.) UNI: g is
// the same in every lane, in a scalar register. The compiler does not see the
// block's instructions: a half is written another instruction after its
// neighbour, and p, whose exp the next instruction could not take, has been read
// by then.
template <bool UNI>
__device__ __forceinline__ void split4(const float (&p)[4], float g, f16x8 &hi, f16x8 &lo, int at) {
    f16x2 h[2];
    uint32_t l[2];
#pragma unroll
    for (int i = 0; i < 2; i++) h[i] = __builtin_convertvector((f32x2){p[2 * i] * g, p[2 * i + 1] * g}, f16x2);
#define REST(G)                                                                                                                      \
    asm("v_fma_mixlo_f16 %0, %2, %6, -%7 op_sel_hi:[0,0,1]\n\t"                                                                      \
        "v_fma_mixlo_f16 %1, %4, %6, -%8 op_sel_hi:[0,0,1]\n\t"                                                                      \
        "v_fma_mixhi_f16 %0, %3, %6, -%7 op_sel:[0,0,1] op_sel_hi:[0,0,1]\n\t"                                                       \
        "v_fma_mixhi_f16 %1, %5, %6, -%8 op_sel:[0,0,1] op_sel_hi:[0,0,1]"                                                           \
        : "=&v"(l[0]), "=&v"(l[1])                                                                                                   \
        : "v"(p[0]), "v"(p[1]), "v"(p[2]), "v"(p[3]), G(g), "v"(h[0]), "v"(h[1]))
    if (UNI) REST("s");
    else REST("v");
#undef REST
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const f16x2 b = __builtin_bit_cast(f16x2, l[i]);
        hi[at + 2 * i] = h[i][0];
        hi[at + 2 * i + 1] = h[i][1];
        lo[at + 2 * i] = b[0];
        lo[at + 2 * i + 1] = b[1];
    }
}

// The largest of two or three; unlike fmaxf's code, operands are taken as they
// are (no signalling NaN reaches here), one instruction each.
__device__ __forceinline__ float max2(float a, float b) {
    float r;
    asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
// Over the wave's four rows of lanes: a swap leaves both partners' values in
// every lane.
__device__ __forceinline__ float rows_max(float m, float v) {
    const uint32_t a = __float_as_uint(v);
    const auto p = __builtin_amdgcn_permlane16_swap(a, a, false, false);
    const uint32_t b = __float_as_uint(max2(__uint_as_float(p[0]), __uint_as_float(p[1])));
    const auto q = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    return max3(m, __uint_as_float(q[0]), __uint_as_float(q[1]));
}

// One group of UN tiles' scores to weights, online: updates the row's maximum and
// sum, gives the weights' f16 halves in operand order and what the output so far
// is to be multiplied by. x: the integer scores; f: what they are to be multiplied
// by (scale, q's unit, the keys' scale), v: the values' scale, per tile. Key `key` + 16 u + 4 lg + e is visible up to pos (groups are aligned,
// so that the sum stays in 32 bits at the last position, too).
// The usual group has all its keys visible, f >= 0, exponents within KV8_FAR and
// the values' scales at least 2^-80, and looks only whether some exponent passes
// the maximum kept. GEN takes any: masked keys apart (a row with no key yet has
// the maximum -inf), whose block's scale, NaN perhaps, is not theirs to see; and
// scores of any size. Next to a far maximum they are rounded before they are
// compared, all in the same way: an unrounded product can lie whole powers of two
// above or below its own rounding. far: some row is, and was taken by GEN.
template <int UN, bool GEN>
__device__ __forceinline__ float softmax_step(const float (&x)[UN][4], const float (&f)[UN], const v_scale (&v)[UN], uint32_t key, uint32_t pos,
                                              float &mrun, float &lsum, bool &far, f16x8 (&ph)[UN / 2], f16x8 (&pl)[UN / 2]) {
    const uint32_t k0 = key + ((threadIdx.x & 63) >> 4 << 2);
    float t[UN][4], al = 1.0f, over;
    auto score = [&](int u, int e) {
        float s = x[u][e] * f[u];
        asm("" : "+v"(s));          // rounded here
        return s;
    };
    auto exponents = [&]() {
#pragma unroll
        for (int u = 0; u < UN; u++)
#pragma unroll
            for (int e = 0; e < 4; e++) t[u][e] = fmaf(x[u][e], f[u], v[u].e - mrun);
    };
    if (!GEN) {
        exponents();
#pragma unroll
        for (int u = 0; u < UN; u++) {
            const float m = max3(t[u][0], t[u][1], t[u][2]);
            over = u ? max3(over, m, t[u][3]) : max2(m, t[u][3]);
        }
    }
    if (GEN || __builtin_amdgcn_ballot_w64(!(over <= KV8_OVER))) {
        float tm = -INFINITY;
#pragma unroll
        for (int u = 0; u < UN; u++) {
            if (GEN) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float m = score(u, e) + v[u].e;
                    tm = fmaxf(tm, k0 + 16 * u + e <= pos ? m : -INFINITY);
                }
            } else {
                tm = max2(tm, fmaf(max2(max3(x[u][0], x[u][1], x[u][2]), x[u][3]), f[u], v[u].e));
            }
        }
        const float mnew = ceilf(rows_max(mrun, tm));
        const float off = GEN ? far_off(mnew) : 0.0f, was = GEN ? far_off(mrun) : 0.0f;
        al = mrun == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((mrun - mnew) + (was - off));
        mrun = mnew;
        lsum *= al;
        exponents();
        if (GEN && __builtin_amdgcn_ballot_w64(off != 0.0f)) {
            far = true;
#pragma unroll
            for (int u = 0; u < UN; u++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float r = (score(u, e) - mrun) + (v[u].e - off);
                    if (off != 0.0f) t[u][e] = r > KV8_OVER ? KV8_OVER : r;
                }
        }
    }
    float l = lsum;
#pragma unroll
    for (int u = 0; u < UN; u++) {
        const float g = GEN && k0 + 16 * u > pos ? 0.0f : v[u].g;
        float p[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            p[e] = __builtin_amdgcn_exp2f(t[u][e]);
            if (GEN && k0 + 16 * u + e > pos) p[e] = 0.0f;
        }
        l = fmaf((p[0] + p[1]) + (p[2] + p[3]), v[u].rs, l);
        split4<!GEN>(p, g, ph[u / 2], pl[u / 2], 4 * (u & 1));
    }
    lsum = l;
    return al;
}

template <int HD, int NW>
__global__ void __launch_bounds__(NW * 64, 2) k_kv8_wave(sgk_kv8_attn a, kv8_part part, int al) {
    constexpr int NC = HD / 64, NT = HD / 16, OLD = HD + 4;
    __shared__ float wm[NW][16], wl[NW][16];
    __shared__ __align__(16) float ob[NW][16 * OLD];
    const uint32_t t = threadIdx.x, lane = t & 63, li = lane & 15, lg = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const uint32_t hk = blockIdx.y, sp = blockIdx.x, S = part.splits.d, G = part.group.d;
    const uint32_t r0 = blockIdx.z * 16, R = min(a.ntok * G - r0, 16u), first = a.base + div_by(r0, part.group);    // first: visible to all rows
    const uint32_t ntile = (a.base + div_by(r0 + R - 1, part.group)) / KV8_T + 1, nstep = (ntile + 1) / 2;
    uint32_t s0, s1;
    part_of(nstep, sp, part.splits, s0, s1);
    const uint32_t bsh = __builtin_ctz(a.block / KV8_T);
    const uint32_t row_of = r0 + min(li, R - 1), tok = div_by(row_of, part.group), head = hk * G + row_of - tok * G, rpos = a.base + tok;
    const int8_t *codes = a.codes + (size_t)hk * (2 * KV8_T * HD) + lane * 16;
    const size_t rec = (size_t)a.n_kv * (2 * KV8_T * HD);
    const float *scales = a.scales + 2 * hk;
    const size_t srec = 2 * (size_t)a.n_kv;

    v4u kr[2][NC], vr[2][NC];
    float ks[2], vs[2], nks[2], nvs[2];
    auto tile_of = [&](uint32_t step, int u) { return min(2 * step + u, ntile - 1); };
    auto load_k = [&](uint32_t step) {
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const v4u *p = (const v4u *)(codes + tile_of(step, u) * rec);
#pragma unroll
            for (int c = 0; c < NC; c++) kr[u][c] = __builtin_nontemporal_load(p + c * 64);
        }
    };
    auto load_v = [&](uint32_t step) {
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const v4u *p = (const v4u *)(codes + tile_of(step, u) * rec + KV8_T * HD);
#pragma unroll
            for (int c = 0; c < NC; c++) vr[u][c] = __builtin_nontemporal_load(p + c * 64);
        }
    };
    auto load_s = [&](uint32_t step) {
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const float *p = scales + (size_t)(tile_of(step, u) >> bsh) * srec;
            nks[u] = p[0];
            nvs[u] = p[1];
        }
    };
    uint32_t step = s0 + wave;
    const bool any = step < s1;
    const q_start start = q_starts();
    v4i qd[3][NC];
    float qf = 0.0f;
    uint32_t kmost = 0;
    if (any) {
        float xq[NC][16];
        q_load<NC>(a.q + tok * a.q_tok + (size_t)head * a.q_stride, al, lg, xq);
        load_s(step);
        load_k(step);
        __builtin_amdgcn_sched_barrier(0);      // all keys, then the values: in the loop's order, whose waits count them
        load_v(step);
        __builtin_amdgcn_sched_barrier(0);
        qf = q_row<NC>(xq, a.scale * 1.44269504088896340736f, qd);
        kmost = __builtin_amdgcn_readfirstlane(__float_as_uint(ks_most(qf, HD)));
    }
    f32x4 o[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) o[n] = (f32x4){0.f, 0.f, 0.f, 0.f};
    float mrun = -INFINITY, lsum = 0.0f;
    bool far = false;
    // The last step stands apart: with its missing loads in the loop, waiting for
    // a step's keys is waiting for its values as well.
    auto work = [&](bool more) {
        float sc[2][4];
#pragma unroll
        for (int u = 0; u < 2; u++) { ks[u] = nks[u]; vs[u] = nvs[u]; }
#pragma unroll
        for (int u = 0; u < 2; u++) {
            v4i s[3] = {start.lo, {0, 0, 0, 0}, start.hi};
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int d = 0; d < 3; d++)
                    s[d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(v4i, kr[u][c]), qd[d][c], s[d], 0, 0, 0);
#pragma unroll
            for (int e = 0; e < 4; e++) sc[u][e] = q_join(s[0][e], s[1][e], s[2][e]);
        }
        if (more) { load_s(step + NW); load_k(step + NW); }
        f16x8 ph[1], pl[1];
        uint32_t kb[2], vb[2];
#pragma unroll
        for (int u = 0; u < 2; u++) {
            kb[u] = __builtin_amdgcn_readfirstlane(__float_as_uint(ks[u]));
            vb[u] = __builtin_amdgcn_readfirstlane(__float_as_uint(vs[u]));
        }
        const float f[2] = {qf * __uint_as_float(kb[0]), qf * __uint_as_float(kb[1])};
        float al2;
        if (step * 32 + 31 <= first && !far && scales_usual(kb[0], vb[0], kmost) && scales_usual(kb[1], vb[1], kmost)) {
            const v_scale v[2] = {v_scale_usual(vb[0]), v_scale_usual(vb[1])};
            al2 = softmax_step<2, false>(sc, f, v, 0, 0, mrun, lsum, far, ph, pl);
        } else {
            const v_scale v[2] = {v_scale_of(vs[0]), v_scale_of(vs[1])};
            al2 = softmax_step<2, true>(sc, f, v, step * 32, rpos, mrun, lsum, far, ph, pl);
        }
        if (step != s0 + wave && __builtin_amdgcn_ballot_w64(al2 != 1.0f)) {       // the first step has nothing to rescale
#pragma unroll
            for (int n = 0; n < NT; n++) o[n] *= al2;
        }
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const f16x8 v = codes_f16(vr[0][c][j], vr[1][c][j]);
                o[4 * c + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, ph[0], o[4 * c + j], 0, 0, 0);
                o[4 * c + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pl[0], o[4 * c + j], 0, 0, 0);
            }
        if (more) load_v(step + NW);
    };
    for (; step + NW < s1; step += NW) work(true);
    if (any) work(false);
    // join the waves: each leaves its maximum, sum and output (-inf and zeros
    // without a step), one barrier. All of a row's are asked for at once.
    if (far) {
        const float k = __builtin_amdgcn_exp2f(far_off(mrun));
        lsum *= k;
#pragma unroll
        for (int n = 0; n < NT; n++) o[n] *= k;
    }
    lsum += swap16f(lsum);
    lsum += swap32f(lsum);
    if (li < R) {
        if (lg == 0) { wm[wave][li] = mrun; wl[wave][li] = lsum; }
        float *dst = &ob[wave][li * OLD + 4 * lg];
#pragma unroll
        for (int n = 0; n < NT; n++) *(f32x4 *)(dst + 16 * n) = o[n];
    }
    __syncthreads();
    for (uint32_t i = t; i < R * (HD / 4); i += NW * 64) {
        const uint32_t r = i / (HD / 4), d = i % (HD / 4) * 4;
        float wmx[NW], m = -INFINITY, l = 0.0f;
        f32x4 ov[NW], v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < NW; w++) { wmx[w] = wm[w][r]; ov[w] = *(const f32x4 *)&ob[w][r * OLD + d]; }
#pragma unroll
        for (int w = 0; w < NW; w++) m = fmaxf(m, wmx[w]);
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const float f = wmx[w] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(wmx[w] - m);
            l = fmaf(wl[w][r], f, l);
            v += ov[w] * f;
        }
        const uint32_t z = div_by(r0 + r, part.group);
        const size_t row = (size_t)z * a.n_heads + hk * G + (r0 + r - z * G);
        if (S == 1) {
            st4(a.out + row * HD + d, v / l, !((uintptr_t)a.out & 15));
        } else {
            *(f32x4 *)(part.acc + (row * S + sp) * HD + d) = v;
            // a sum that is NaN has to reach the join whatever the maximum
            if (d == 0) { part.m[row * S + sp] = l != l ? 0.0f : m; part.s[row * S + sp] = l; }
        }
    }
}

// ---------------------------------------------------------------------------
// Attention of many rows: a workgroup takes 128 consecutive rows, 16 to a wave
// (token-major, the query heads of one kv head inside a token, so any group
// size fills them), and walks its keys in tiles of 64, staged once in LDS for
// all of them: the key codes as they lie (1 KB per operand fragment, 16 bytes
// a lane, no bank conflict), the value codes turned into f16 on the way. The
// arithmetic is the wave form's.
// A tile's work for a wave is 112 matrix products of 16 cycles (head_dim 256)
// and about 240 vector instructions. Waves that run both in step leave the
// matrix unit idle through the softmax: 46% busy. So the two waves of a SIMD (w
// and w + 4) alternate: one is in its products (the last tile's P V, this one's
// K Q^T) while the other is in its softmax, with a barrier a tile. Beside a
// wave that keeps the matrix unit busy another issues two vector instructions
// per product (measured), so 224 products and 480 of those take at least 3800
// cycles, of which 3584 are the products'; over a launch it is busy 63%.
// Both tiles are double-buffered; a wave stores its part of the next one and
// requests that of the one after before its softmax.
// 24 heads of 256 on 4, 2048 tokens at 14336: 980-1050 us, 770 TFLOP/s of the
// formula's, and as the matrix unit counts them (weights in two halves, three
// digits at twice the rate) 1340, where a plain f16 product of 16384^3 reaches
// 1346: the clock falls to 1.7 GHz under the load. At head_dim 128 and 64 the
// vector instructions bound it: 216 and 204 for 56 and 28 products.
// Grid: (row block, kv head, key split), the longest rows first.
// ---------------------------------------------------------------------------
#define KV8_NW 8
#define KV8_ROWS (KV8_NW * 16u)

// LDS done, then the barrier; loads from memory stay in flight
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// head_dim 64 stays within the 128 registers that let a second workgroup in (12 of
// 64, 4096 tokens at 8192: 356 us, with one 439); a row's place, two registers,
// lies in memory through the loops.
template <int HD>
__global__ void __launch_bounds__(KV8_NW * 64, HD == 64 ? 4 : 2) k_kv8_tile(sgk_kv8_attn a, kv8_part part, int al) {
    constexpr int NC = HD / 64, NT = HD / 16, NTH = KV8_NW * 64;
    constexpr int KCH = 4 * NC * 64, VUN = 2 * NC * 64;     // 16-byte chunks of keys, units (two chunks) of values
    constexpr int KPT = (KCH + NTH - 1) / NTH, VPT = (VUN + NTH - 1) / NTH;
    __shared__ v4u kb[2][KCH];
    __shared__ v4u vb[2][2 * NT * 64];
    const uint32_t t = threadIdx.x, lane = t & 63, li = lane & 15, lg = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const uint32_t hk = blockIdx.y, sp = blockIdx.z, S = part.splits.d, G = part.group.d;
    const uint64_t R = (uint64_t)a.ntok * G, r0 = (uint64_t)(gridDim.x - 1 - blockIdx.x) * KV8_ROWS;
    const uint32_t lastk = a.base + div_by((uint32_t)(min(r0 + KV8_ROWS, R) - 1), part.group);      // the block's last visible key
    const uint32_t nrec = lastk / KV8_T + 1, nt = lastk / 64 + 1;
    uint32_t k0, k1;
    part_of(nt, sp, part.splits, k0, k1);
    const uint32_t n = k1 - k0;             // tiles k0 .. k0 + n - 1
    const uint32_t bsh = __builtin_ctz(a.block / KV8_T);
    const size_t rec = (size_t)a.n_kv * (2 * KV8_T * HD);
    const int8_t *codes = a.codes + (size_t)hk * (2 * KV8_T * HD);
    const float *scales = a.scales + 2 * hk;
    const size_t srec = 2 * (size_t)a.n_kv;

    // This thread's chunks of a tile (counted from k0): a uniform address and an
    // offset of its own, computed again only in the tile that the cache's end
    // cuts. Every thread loads (chunks past the tile's are its first again),
    // so that no wait for one load has to cover the next.
    v4u kr[KPT], vr[VPT][2];
    const uint32_t rec32 = (uint32_t)rec;       // a record row is at most 2^29 bytes
    uint32_t koff[KPT], voff[VPT];
    auto k_at = [&](uint32_t t, int x, uint32_t last) {
        const uint32_t c = (t + x * NTH) % KCH;
        return min(c / (NC * 64), last) * rec32 + c % (NC * 64) * 16;
    };
    auto v_at = [&](uint32_t t, int x, int j, uint32_t last) {
        const uint32_t c = (t + x * NTH) % VUN;
        return min(c / (NC * 64) * 2 + j, last) * rec32 + c % (NC * 64) * 16 + KV8_T * HD;
    };
#pragma unroll
    for (int x = 0; x < KPT; x++) koff[x] = k_at(t, x, 3);
#pragma unroll
    for (int x = 0; x < VPT; x++) voff[x] = v_at(t, x, 0, 3);
    auto load_k = [&](uint32_t i) {
        const uint32_t r4 = 4 * (k0 + i), last = nrec - 1 - r4;     // records from the tile's first that exist
        const int8_t *p = codes + (size_t)r4 * rec;
        uint32_t at[KPT];
#pragma unroll
        for (int x = 0; x < KPT; x++) at[x] = koff[x];
        if (last < 3) {
            uint32_t tc = t;
            asm volatile("" : "+v"(tc));            // here and now, not in registers through the loop
#pragma unroll
            for (int x = 0; x < KPT; x++) at[x] = k_at(tc, x, last);
        }
#pragma unroll
        for (int x = 0; x < KPT; x++) kr[x] = *(const v4u *)(p + at[x]);
    };
    auto load_v = [&](uint32_t i) {
        const uint32_t r4 = 4 * (k0 + i), last = nrec - 1 - r4;
        const int8_t *p = codes + (size_t)r4 * rec;
        uint32_t at[VPT][2];
#pragma unroll
        for (int x = 0; x < VPT; x++) { at[x][0] = voff[x]; at[x][1] = voff[x] + rec32; }
        if (last < 3) {
            uint32_t tc = t;
            asm volatile("" : "+v"(tc));
#pragma unroll
            for (int x = 0; x < VPT; x++)
#pragma unroll
                for (int j = 0; j < 2; j++) at[x][j] = v_at(tc, x, j, last);
        }
#pragma unroll
        for (int x = 0; x < VPT; x++)
#pragma unroll
            for (int j = 0; j < 2; j++) vr[x][j] = *(const v4u *)(p + at[x][j]);
    };
    // A tile's scales, one to a lane: lane j holds record j % 4's of its keys (j
    // / 4 % 2 == 0) or values. 4 T >> bsh plus j >> bsh is (4 T + j) >> bsh.
    const uint32_t soff = ((lane & 3) >> bsh) * (uint32_t)srec + (lane >> 2 & 1);
    float sn;
    auto load_s = [&](uint32_t i) {
        const uint32_t r4 = 4 * (k0 + i), last = nrec - 1 - r4;
        uint32_t at = soff;
        if (last < 3) {
            uint32_t lc = lane;
            asm volatile("" : "+v"(lc));
            at = (min(lc & 3, last) >> bsh) * (uint32_t)srec + (lc >> 2 & 1);
        }
        sn = (scales + (size_t)(r4 >> bsh) * srec)[at];
    };
    auto stage_k = [&](uint32_t i) {
#pragma unroll
        for (int x = 0; x < KPT; x++) {
            const uint32_t c = t + x * NTH;
            if (KCH % NTH == 0 || wave * 64 + x * NTH < KCH) kb[i & 1][c] = kr[x];
        }
    };
    auto stage_v = [&](uint32_t i) {
#pragma unroll
        for (int x = 0; x < VPT; x++) {
            const uint32_t c = t + x * NTH;
            if (VUN % NTH == 0 || wave * 64 + x * NTH < VUN)
#pragma unroll
                for (int j = 0; j < 4; j++)         // fragment (pair of tiles, dims 16 (4 c + j) ..)
                    vb[i & 1][(c / 64 * 4 + j) * 64 + c % 64] = __builtin_bit_cast(v4u, codes_f16(vr[x][0][j], vr[x][1][j]));
        }
    };

    const uint64_t r = r0 + wave * 16 + li, rw = r0 + wave * 16;
    const uint32_t tok = r < R ? div_by((uint32_t)r, part.group) : 0, head = hk * G + (r < R ? (uint32_t)r - tok * G : 0), rpos = a.base + tok;
    float xq[NC][16];
    q_load<NC>(a.q + tok * a.q_tok + (size_t)head * a.q_stride, al, lg, xq);
    if (n) load_k(0);
    v4i qd[3][NC];
    const float qf = q_row<NC>(xq, a.scale * 1.44269504088896340736f, qd);
    // the usual scales' bounds, keys' or values' as in sn
    const float least = lane & 4 ? 0x1p-80f : 0.0f, most = lane & 4 ? 0x1.fffffep127f : ks_most(qf, HD);
    const q_start start = q_starts();
    float mrun = -INFINITY, lsum = 0.0f, resc = 1.0f;
    bool far = false;
    f32x4 o[NT];
#pragma unroll
    for (int d = 0; d < NT; d++) o[d] = (f32x4){0.f, 0.f, 0.f, 0.f};
    // the wave's first and last visible keys: no mask up to the one, no work past the other
    const uint32_t wfirst = a.base + div_by((uint32_t)rw, part.group);
    const uint32_t wtiles = rw < R ? (a.base + div_by((uint32_t)(min(rw + 16, R) - 1), part.group)) / 64 + 1 : 0;
    const uint32_t ntw = wtiles > k0 ? min(wtiles - k0, n) : 0;
    float sc[4][4];
    f16x8 ph[2], pl[2];
    // Step of products, tile i: P V of tile i - 1, K Q^T of tile i. The other
    // wave of the SIMD is in its softmax, so the wave has to cover the LDS reads
    // itself: fragments go through a ring of five, each requested four ahead (8
    // products, 128 cycles), and the two halves of a P V pair are two
    // products apart. At the ends it multiplies zeros (no tile -1: its weights
    // and values are) or what nobody reads (no tile n).
    auto products = [&](uint32_t i) {
        constexpr int NV = 2 * NT, NK = 4 * NC, RING = 5;
        const v4u *vt = vb[(i + 1) & 1] + lane, *kt = kb[i & 1] + lane;
        v4u fr[RING];
        auto fetch = [&](int k) {
            if (k < NV + NK) fr[k % RING] = k < NV ? vt[k * 64] : kt[(k - NV) * 64];
        };
#pragma unroll
        for (int k = 0; k < RING - 1; k++) fetch(k);
        if (__builtin_amdgcn_ballot_w64(resc != 1.0f)) {
#pragma unroll
            for (int d = 0; d < NT; d++) o[d] *= resc;
        }
#pragma unroll
        for (int k = 0; k <= NV; k++) {
            if (k) o[(k - 1) % NT] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, fr[(k - 1) % RING]), pl[(k - 1) / NT],
                                                                            o[(k - 1) % NT], 0, 0, 0);
            if (k < NV) o[k % NT] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, fr[k % RING]), ph[k / NT], o[k % NT], 0, 0, 0);
            if (k < NV) fetch(k + RING - 1);
            __builtin_amdgcn_sched_barrier(0);
        }
        // A record's scores are joined behind the next one's first products, in this
        // order (left to the compiler, joins that wait for their products come
        // between: 24 heads of 256 on 4, 2048 tokens at 14336 1007 us against 1040 to
        // 1130, 32 of 128 on 8 807 against 900); at head_dim 64, with one product a
        // sum, as they come (12 heads 368 against 388).
        constexpr bool LATE = NC > 1;
        v4i s[2][3];
        auto join = [&](int u) {
#pragma unroll
            for (int e = 0; e < 4; e++) sc[u][e] = q_join(s[u & 1][0][e], s[u & 1][1][e], s[u & 1][2][e]);
        };
#pragma unroll
        for (int k = 0; k < NK; k++) {
            const int u = k / NC, c = k % NC;
            if (c == 0) { s[u & 1][0] = start.lo; s[u & 1][1] = (v4i){0, 0, 0, 0}; s[u & 1][2] = start.hi; }
#pragma unroll
            for (int d = 0; d < 3; d++)
                s[u & 1][d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(v4i, fr[(NV + k) % RING]), qd[d][c], s[u & 1][d], 0, 0, 0);
            fetch(NV + k + RING - 1);
            if (LATE ? u && c == 1 : c == NC - 1) join(LATE ? u - 1 : u);
            if (LATE) __builtin_amdgcn_sched_barrier(0);
        }
        if (LATE) join(3);
    };
    auto weights = [&](uint32_t i) {
        auto from = [](float v, int j) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), j)); };
        const uint32_t key = (k0 + i) * 64;
        const float f[4] = {qf * from(sn, 0), qf * from(sn, 1), qf * from(sn, 2), qf * from(sn, 3)};
        const v_scale s = v_scale_of(sn);
        const v_scale v[4] = {{from(s.e, 4), from(s.g, 4), from(s.rs, 4)}, {from(s.e, 5), from(s.g, 5), from(s.rs, 5)},
                              {from(s.e, 6), from(s.g, 6), from(s.rs, 6)}, {from(s.e, 7), from(s.g, 7), from(s.rs, 7)}};
        if (key + 63 <= wfirst && !far && !__builtin_amdgcn_ballot_w64(__builtin_amdgcn_fmed3f(sn, least, most) != sn))
            resc = softmax_step<4, false>(sc, f, v, 0, 0, mrun, lsum, far, ph, pl);
        else
            resc = softmax_step<4, true>(sc, f, v, key, rpos, mrun, lsum, far, ph, pl);
    };

    ph[0] = ph[1] = pl[0] = pl[1] = (f16x8){};
#pragma unroll
    for (int x = 0; x < 2 * NT * 64; x += NTH)
        if (2 * NT * 64 % NTH == 0 || t + x < 2 * NT * 64) vb[1][t + x] = (v4u){0, 0, 0, 0};
    if (n) {
        stage_k(0);
        load_k(min(1u, n - 1));
        load_v(0);
        load_s(0);
    }
    lds_barrier();
    // Period i (two steps, one barrier): group 0 does the products of tile i and
    // the softmax of i, group 1 the softmax of i - 1 and the products of i. Read
    // are the keys of tile i and the values of i - 1; written, in a wave's
    // softmax step, the keys of i + 1 and the values of i, requested a period ago.
    // Past the last tile it stages that one again, where nobody reads it.
    // A loop for each group: with the two orders in one the compiler keeps the
    // state of both at the branch, 60 moves a step and a wait for the loads.
    auto soften = [&](uint32_t next, int i) {
        stage_k(next + 1);
        stage_v(next);
        load_k(min(next + 2, n - 1));
        load_v(min(next + 1, n - 1));
        if (i >= 0 && (uint32_t)i < ntw) {
            weights(i);
        } else {
            ph[0] = ph[1] = pl[0] = pl[1] = (f16x8){};
            resc = 1.0f;
        }
        load_s(min((uint32_t)(i + 1), n - 1));
    };
    if (n && wave < KV8_NW / 2) {
        for (uint32_t i = 0; i <= n; i++) {
            products(i);
            soften(i, (int)i);
            lds_barrier();
        }
    } else if (n) {
        for (uint32_t i = 0; i <= n; i++) {
            soften(i, (int)i - 1);
            products(i);
            lds_barrier();
        }
    }
    if (far) {
        const float k = __builtin_amdgcn_exp2f(far_off(mrun));
        lsum *= k;
#pragma unroll
        for (int n = 0; n < NT; n++) o[n] *= k;
    }
    lsum += swap16f(lsum);
    lsum += swap32f(lsum);
    if (r >= R) return;
    const float l = lsum;
    const size_t row = (size_t)tok * a.n_heads + head;
    if (S == 1) {
        const bool oal = !((uintptr_t)a.out & 15);
#pragma unroll
        for (int d = 0; d < NT; d++) st4(a.out + row * HD + 16 * d + 4 * lg, o[d] / l, oal);
    } else {
        float *acc = part.acc + (row * S + sp) * HD + 4 * lg;
#pragma unroll
        for (int d = 0; d < NT; d++) *(f32x4 *)(acc + 16 * d) = o[d];
        if (lg == 0) { part.m[row * S + sp] = l != l ? 0.0f : mrun; part.s[row * S + sp] = l; }
    }
}

// Join of few splits of many rows: four dims of a row per lane, all splits'
// loads in flight, nothing shared between lanes (49152 rows of 256, two splits,
// 151 MB: 23 us). Every row sees key 0, so the
// largest maximum is a number, and a split without a key weighs nothing; NaN
// sums reach the output.
#define KV8_JOIN 8u
template <int HD>
__global__ void __launch_bounds__(TPB) k_kv8_join(kv8_part p, float *out, uint64_t rows, uint32_t S, int al) {
    constexpr uint32_t L = HD / 4;
    const uint64_t row = (uint64_t)blockIdx.x * (TPB / L) + threadIdx.x / L;
    const uint32_t d = threadIdx.x % L * 4;
    if (row >= rows) return;
    f32x4 acc[KV8_JOIN];
    float m[KV8_JOIN], l[KV8_JOIN], M = -INFINITY, sum = 0.0f;
#pragma unroll
    for (uint32_t k = 0; k < KV8_JOIN; k++) {
        const bool on = k < S;
        m[k] = on ? p.m[row * S + k] : -INFINITY;
        l[k] = on ? p.s[row * S + k] : 0.0f;
        acc[k] = on ? *(const f32x4 *)(p.acc + (row * S + k) * HD + d) : (f32x4){0.f, 0.f, 0.f, 0.f};
        M = fmaxf(M, m[k]);
    }
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (uint32_t k = 0; k < KV8_JOIN; k++) {
        const float w = m[k] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[k] - M);
        sum = fmaf(l[k], w, sum);
        o += acc[k] * w;
    }
    st4(out + row * HD + d, o / sum, al);
}

// Join of many splits of few rows: a workgroup per row and 64 dims, 16 lanes of
// four dims for every 16th split; the first four splits of a lane are asked
// for before the weights. Bound by that chain: 24 rows of 256, 64 splits 4.1 us.
#define KV8_COMB 512u
__global__ void __launch_bounds__(TPB) k_kv8_comb(kv8_part p, float *out, uint32_t hd, uint32_t S, int al) {
    __shared__ float wt[KV8_COMB], red[4], sum[4];
    __shared__ f32x4 pt[16][16];
    const uint32_t t = threadIdx.x, lane = t & 15, g = t >> 4, d = blockIdx.y * 64 + lane * 4;
    const size_t row = blockIdx.x, at = row * S;
    const f32x4 *acc = (const f32x4 *)(p.acc + at * hd + d);
    const uint32_t step = hd / 4;
    f32x4 v[4];
#pragma unroll
    for (int u = 0; u < 4; u++) v[u] = g + 16 * u < S ? acc[(size_t)(g + 16 * u) * step] : (f32x4){0.f, 0.f, 0.f, 0.f};
    float m[KV8_COMB / TPB], l[KV8_COMB / TPB], M = -INFINITY;
#pragma unroll
    for (uint32_t x = 0; x < KV8_COMB / TPB; x++) {
        const uint32_t k = t + x * TPB;
        m[x] = k < S ? p.m[at + k] : -INFINITY;
        l[x] = k < S ? p.s[at + k] : 0.0f;
        M = fmaxf(M, m[x]);
    }
    M = wave_fmax(M);
    if ((t & 63) == 0) red[t >> 6] = M;
    __syncthreads();
    M = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    float L = 0.0f;
#pragma unroll
    for (uint32_t x = 0; x < KV8_COMB / TPB; x++) {
        const float w = m[x] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[x] - M);
        if (t + x * TPB < S) wt[t + x * TPB] = w;
        L = fmaf(l[x], w, L);
    }
    L = wave_fsum(L);
    if ((t & 63) == 0) sum[t >> 6] = L;
    __syncthreads();
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < 4; u++)
        if (g + 16 * u < S) o += v[u] * wt[g + 16 * u];
    for (uint32_t k = g + 64; k < S; k += 16) o += acc[(size_t)k * step] * wt[k];
    pt[g][lane] = o;
    __syncthreads();
    if (t >= 16) return;
    o = pt[0][t];
#pragma unroll
    for (int x = 1; x < 16; x++) o += pt[x][t];
    st4(out + row * hd + d, o / ((sum[0] + sum[1]) + (sum[2] + sum[3])), al);
}

// How a call runs. The wave form, small calls (whole calls below in us):
//  - one workgroup of eight waves for 5 to 24 steps of 32 keys (20 at head_dim
//    256), as a second launch to join costs more than a wave's second and third
//    step (one / splits of four waves: 384 keys, 24 heads of 256 on 4 17.2 / 19.1,
//    32 of 128 on 8 14.9 / 17.0, 12 of 64 13.6 / 15.4; 640 keys 19.2 / 19.3, 15.9 /
//    17.0, 14.6 / 15.6; 768 keys 20.8 / 19.3, 16.7 / 17.1, 15.0 / 15.8);
//  - else parts of the keys, one workgroup a CU (two at head_dim 64) of four
//    waves, which spend less on their start and join (four / eight: 24 of 256 on
//    4, 32771 keys 27.4 / 27.8, 5 tokens at 40000 34.6 / 36.3; 32 of 128 on 8, 32771
//    keys 25.3 / 26.0; two workgroups a CU of four 30.3, 45.2, 28.3);
//  - of eight below head_dim 256 where a CU has more than 64 steps, which its
//    vector units and not the cache's bytes bound then (32 of 128 on 8, 40 tokens
//    at 8000 33.3 / 31.4, 20 at 32000 49.0 / 44.3, 262000 keys 96.0 / 95.3).
// Else row blocks in tiles, one workgroup per CU at a time (head_dim 64 has room
// for two), their keys split where that shortens the launch: rounds x (a part's
// tiles + KV8_TAIL for its start and end) tiles of KV8_TILE_US, against the
// partials' way to memory and back. A tile's time is measured at head_dim 256 and
// taken as proportional; at 128 and 64 it is 1.6-1.7 and 1.4 us, so that the rule
// splits less there than it could. KV8_SMALL, in waves' steps of 32 keys x head_dim, is where the two meet
// (wave / tile): 24 heads of 256 on 4, 8040 keys, 240 rows (3.9M) 39.4 / 45.2,
// 1300 keys, 1800 rows (4.7M) 38.1 / 48.2, 8077 keys, 462 rows (7.5M) 53.8 /
// 55.2, 32020 keys, 120 rows (8.2M) 55.7 / 54.0; 32 of 128 on 8, 8040 keys, 160
// rows (2.6M) 30.9 / 38.6, 32020 keys, 80 rows (5.1M) 43.7 / 49.6, 8077 keys, 308
// rows (5.2M) 50.5 / 48.2; 12 of 64, 32077 keys, 77 rows (3.9M) 43.3 / 54.4.
#define KV8_SMALL (5ull << 20)
#define KV8_TILE_US 2.5         /* at head_dim 256 */
#define KV8_TAIL 3.0
#define KV8_PART_BYTES (256ull << 20)
struct kv8_plan { uint32_t waves, splits, blocks; };     // waves: of a workgroup of the wave form, 0 for tiles
static kv8_plan kv8_plan_of(const sgk_kv8_attn *a) {
    const uint64_t G = a->n_heads / a->n_kv, rows = a->ntok * G, keys = (uint64_t)a->base + a->ntok, cus = sgk_device_cus();
    const bool wave = rows <= 16 || (rows + 15) / 16 * a->n_kv * ((keys + 31) / 32) * a->hd <= KV8_SMALL;
    const uint64_t per = wave ? 16 : KV8_ROWS, wgs = (rows + per - 1) / per * a->n_kv;
    kv8_plan p = {wave ? 4u : 0u, 1, (uint32_t)((rows + per - 1) / per)};
    if (wave) {
        const uint64_t steps = (keys + 31) / 32;
        uint64_t most = (a->hd == 64 ? 2 : 1) * cus / wgs;
        if (most > KV8_COMB) most = KV8_COMB;
        const bool one = steps > 4 && steps <= (a->hd == 256 ? 20 : 24);
        if (most && (one || (a->hd < 256 && wgs * steps > 64 * cus))) {
            p.waves = 8;
            p.splits = one ? 1 : (uint32_t)most;
        } else if (most > 1) {
            p.splits = (uint32_t)((steps + 3) / 4 < most ? (steps + 3) / 4 : most);
        }
        return p;
    }
    const uint64_t tiles = (keys + 63) / 64, prow = (uint64_t)a->ntok * a->n_heads * a->hd * 4;
    uint64_t most = wgs < cus ? 2 * cus / wgs : KV8_JOIN;
    if (most > KV8_COMB) most = KV8_COMB;
    if (most > tiles) most = tiles;
    double best = 0.0;
    for (uint64_t S = 1; S <= most && (S == 1 || S * prow <= KV8_PART_BYTES); S++) {
        const double rounds = (double)((wgs * S + cus - 1) / cus), part = (double)((tiles + S - 1) / S) + KV8_TAIL;
        const double cost = rounds * part * KV8_TILE_US * a->hd / 256 + (S > 1 ? 5.0 + (double)(2 * S * prow) / 4.0e6 : 0.0);
        if (S == 1 || cost < best) { best = cost; p.splits = (uint32_t)S; }
    }
    return p;
}

extern "C" uint32_t sgk_kv8_attn_parts(const sgk_kv8_attn *a, uint32_t *waves) {
    const kv8_plan p = kv8_plan_of(a);
    if (waves) *waves = p.waves;
    return p.splits;
}
extern "C" uint64_t sgk_kv8_attn_scratch(const sgk_kv8_attn *a) {
    const kv8_plan p = kv8_plan_of(a);
    return p.splits > 1 ? (uint64_t)a->ntok * a->n_heads * p.splits * (a->hd + 2) * 4 : 0;
}

extern "C" hipError_t sgk_kv8_attention(const sgk_kv8_attn *a, void *scratch, hipStream_t s, hipEvent_t done) {
    if (!a->ntok || !a->n_heads) return hipSuccess;
    if (!sgk_kv8_shape_ok(a->n_kv, a->hd, a->block) || ((uintptr_t)a->codes & 15) || a->n_heads % a->n_kv ||
        a->n_heads / a->n_kv > SGK_KV8_MAX_GROUP) return hipErrorInvalidValue;
    const kv8_plan p = kv8_plan_of(a);
    if (p.splits > 1 && !scratch) return hipErrorInvalidValue;
    const int al = !((uintptr_t)a->q & 15) && a->q_stride % 4 == 0 && a->q_tok % 4 == 0;
    const uint64_t rows = (uint64_t)a->ntok * a->n_heads * p.splits;
    kv8_part part = {};
    part.group = kv8_div_of(a->n_heads / a->n_kv);
    part.splits = kv8_div_of(p.splits);
    if (p.splits > 1) {                 // outputs first, as they are stored 16 bytes at a time
        part.acc = (float *)scratch;
        part.m = part.acc + rows * a->hd;
        part.s = part.m + rows;
    }
    const dim3 wgrid(p.splits, a->n_kv, p.blocks);
    const hipEvent_t ev = p.splits > 1 ? NULL : done;
#define KC(H)                                                                                                     \
    do {                                                                                                          \
        if (p.waves == 8) launch(k_kv8_wave<H, 8>, wgrid, 512, s, ev, *a, part, al);                              \
        else if (p.waves) launch(k_kv8_wave<H, 4>, wgrid, 256, s, ev, *a, part, al);                              \
        else launch(k_kv8_tile<H>, dim3(p.blocks, a->n_kv, p.splits), KV8_NW * 64, s, ev, *a, part, al);          \
    } while (0)
    switch (a->hd) {
    case 64: KC(64); break;
    case 128: KC(128); break;
    default: KC(256); break;
    }
#undef KC
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.splits == 1) return e;
    const uint64_t n = (uint64_t)a->ntok * a->n_heads, per = TPB / (a->hd / 4);
    const int oal = !((uintptr_t)a->out & 15);
    if (p.splits > KV8_JOIN) {
        launch(k_kv8_comb, dim3((uint32_t)n, a->hd / 64), TPB, s, done, part, a->out, a->hd, p.splits, oal);
        return hipGetLastError();
    }
    const dim3 grid((uint32_t)((n + per - 1) / per));
    switch (a->hd) {
    case 64: launch(k_kv8_join<64>, grid, TPB, s, done, part, a->out, n, p.splits, oal); break;
    case 128: launch(k_kv8_join<128>, grid, TPB, s, done, part, a->out, n, p.splits, oal); break;
    default: launch(k_kv8_join<256>, grid, TPB, s, done, part, a->out, n, p.splits, oal); break;
    }
    return hipGetLastError();
}
