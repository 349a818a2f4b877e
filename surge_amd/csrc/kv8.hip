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

// ---------------------------------------------------------------------------
// Store. One workgroup per (block, kv head, half) holds the block's new rows
// in registers: one read for the maximum and the codes. A unit is 16 elements,
// a row's 16 dims for keys (one 16-byte code store) or 4 positions x 4 dims for
// values (four dwords, transposed in registers); U units per thread.
// Rows before base keep their codes unless the scale grows.
// ---------------------------------------------------------------------------
struct kv8_store_args {
    const float *x[2];
    int8_t *codes;
    float *scales;
    uint64_t stride;
    uint32_t n_kv, hd, block, base, n;
};

// x / s to the nearest integer, ties to even, decided exactly: q = rint(x * (1/s))
// is within one of it, and the remainder x - q s is exact in one fma.
__device__ __forceinline__ int quant(float x, float s, float inv) {
    float q = rintf(x * inv);
    const float r = fmaf(-q, s, x), a = 2.0f * fabsf(r);
    if (a > s || (a == s && ((int)q & 1))) q += copysignf(1.0f, r);
    return (int)fminf(fmaxf(q, -127.0f), 127.0f);
}
__device__ __forceinline__ int8_t requant(int8_t c, double was, double s) {
    return (int8_t)rint((double)c * was / s);
}

template <int U>
__global__ void __launch_bounds__(TPB) k_kv8_store(kv8_store_args a, int al) {
    __shared__ uint32_t red[4];
    const uint32_t t = threadIdx.x, h = blockIdx.y, half = blockIdx.z, hd = a.hd;
    const uint32_t blk = a.base / a.block + blockIdx.x, p0 = blk * a.block;
    const uint32_t lo = max(p0, a.base), hi = (uint32_t)min((uint64_t)p0 + a.block, (uint64_t)a.base + a.n);
    const uint32_t kept = lo - p0, rows = hi - p0;      // rows kept .. rows-1 of the block are new
    const uint32_t units = a.block * hd / 16, d4 = hd / 4, d16 = hd / 16;
    const float *x = a.x[half] + (size_t)(lo - a.base) * a.stride + (size_t)h * hd;
    float *sp = a.scales + ((size_t)blk * a.n_kv + h) * 2 + half;
    const float was = kept ? *sp : 0.0f;
    f32x4 v[U][4];
    uint32_t mx = 0;
#pragma unroll
    for (int u = 0; u < U; u++) {
        const uint32_t i = t + u * TPB;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint32_t r = half ? i / d4 * 4 + j : i / d16, d = half ? i % d4 * 4 : i % d16 * 16 + 4 * j;
            v[u][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
            if (i < units && r >= kept && r < rows) v[u][j] = ld4(x + (size_t)(r - kept) * a.stride + d, al);
#pragma unroll
            for (int e = 0; e < 4; e++) mx = max(mx, __float_as_uint(v[u][j][e]) & 0x7FFFFFFFu);
        }
    }
    mx = wave_umax(mx);
    if ((t & 63) == 0) red[t >> 6] = mx;
    __syncthreads();
    mx = max(max(red[0], red[1]), max(red[2], red[3]));
    // 65520 and above round to infinity in f16; NaN's bits are above those
    const bool poison = mx >= 0x477FF000u || was != was;
    float s = fmaxf(__uint_as_float(poison ? 0 : mx) * (1.0f / 127.0f), poison ? 0.0f : was);
    const bool grew = kept && s > was && !poison;
    if (t == 0) *sp = poison ? NAN : s;
    // a scale near the end of the range: x / s is the same for both times 2^64
    const float up = s < 0x1p-60f ? 0x1p64f : 1.0f, sq = s * up, inv = s > 0.0f ? 1.0f / sq : 0.0f;
    const bool zero = poison || s == 0.0f;
#pragma unroll
    for (int u = 0; u < U; u++) {
        const uint32_t i = t + u * TPB;
        if (i >= units) continue;
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            uint32_t c = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) c |= (uint32_t)(zero ? 0 : quant(v[u][j][e] * up, sq, inv) & 0xFF) << (8 * e);
            w[j] = c;
        }
        if (!half) {
            const uint32_t r = i / d16, d = i % d16 * 16;
            if (r >= rows || (r < kept && !grew)) continue;
            int8_t *p = a.codes + rec_at((p0 + r) / KV8_T, a.n_kv, h, hd) + key_at(r % KV8_T, d);
            if (r < kept) {
                v4u old = *(const v4u *)p;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    uint32_t c = 0;
#pragma unroll
                    for (int e = 0; e < 4; e++) c |= (uint32_t)(requant((int8_t)(old[j] >> (8 * e)), was, s) & 0xFF) << (8 * e);
                    w[j] = c;
                }
            }
            *(v4u *)p = (v4u){w[0], w[1], w[2], w[3]};
        } else {
            const uint32_t r = i / d4 * 4, d = i % d4 * 4;
            if (r >= rows || (r + 4 <= kept && !grew)) continue;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                uint32_t *p = (uint32_t *)(a.codes + a.hd * KV8_T + rec_at((p0 + r) / KV8_T, a.n_kv, h, hd) + val_at(r % KV8_T, d + e));
                uint32_t c = 0;
#pragma unroll
                for (int j = 0; j < 4; j++) c |= (w[j] >> (8 * e) & 0xFF) << (8 * j);
                if (r < kept || r + 4 > rows) {     // some of the four rows are not new
                    const uint32_t old = *p;
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        if (r + j >= kept && r + j < rows) continue;
                        const int8_t o = (int8_t)(old >> (8 * j));
                        const uint32_t b = (uint32_t)(uint8_t)(r + j < kept && grew ? requant(o, was, s) : o);
                        c = (c & ~(0xFFu << (8 * j))) | b << (8 * j);
                    }
                }
                *p = c;
            }
        }
    }
}

extern "C" hipError_t sgk_kv8_store(const float *k, const float *v, uint64_t stride, int8_t *codes, float *scales,
                                    uint32_t n_kv, uint32_t hd, uint32_t block, uint32_t base, uint32_t n, hipStream_t s) {
    if (!n) return hipSuccess;
    if (!sgk_kv8_shape_ok(n_kv, hd, block) || ((uintptr_t)codes & 15)) return hipErrorInvalidValue;
    kv8_store_args a = {{k, v}, codes, scales, stride, n_kv, hd, block, base, n};
    const int al = !((uintptr_t)k & 15) && !((uintptr_t)v & 15) && stride % 4 == 0;
    const uint32_t blocks = (uint32_t)(((uint64_t)base + n + block - 1) / block) - base / block;
    const dim3 grid(blocks, n_kv, 2);
    const uint32_t units = block * hd / 16;
#define SC(U) hipLaunchKernelGGL(k_kv8_store<U>, grid, dim3(TPB), 0, s, a, al)
    if (units <= TPB) SC(1);
    else if (units <= 2 * TPB) SC(2);
    else if (units <= 4 * TPB) SC(4);
    else SC(8);
#undef SC
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Load: a workgroup per (tile, kv head, half), a thread per unit as above.
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(TPB) k_kv8_load(const int8_t *codes, const float *scales, float *k, float *v,
                                                  uint64_t stride, uint32_t n_kv, uint32_t hd, uint32_t block,
                                                  uint32_t base, uint32_t n, int al) {
    const uint32_t tile = base / KV8_T + blockIdx.x, h = blockIdx.y, half = blockIdx.z, i = threadIdx.x;
    if (i >= hd) return;                                // 16 hd / 16 units
    const float s = scales[((size_t)(tile * KV8_T / block) * n_kv + h) * 2 + half];
    const int8_t *rec = codes + rec_at(tile, n_kv, h, hd) + (size_t)half * KV8_T * hd;
    const uint64_t p0 = (uint64_t)tile * KV8_T;
    uint32_t w[4];
    if (!half) {
        const uint32_t r = i % 16, d = i / 16 * 16;
        const v4u q = *(const v4u *)(rec + key_at(r, d));
        if (p0 + r < base || p0 + r >= (uint64_t)base + n) return;
        float *o = k + (size_t)(p0 + r - base) * stride + (size_t)h * hd + d;
#pragma unroll
        for (int j = 0; j < 4; j++)
            st4(o + 4 * j, (f32x4){(int8_t)q[j] * s, (int8_t)(q[j] >> 8) * s, (int8_t)(q[j] >> 16) * s, (int8_t)(q[j] >> 24) * s}, al);
    } else {
        const uint32_t r = i / (hd / 4) * 4, d = i % (hd / 4) * 4;
#pragma unroll
        for (int e = 0; e < 4; e++) w[e] = *(const uint32_t *)(rec + val_at(r, d + e));
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (p0 + r + j < base || p0 + r + j >= (uint64_t)base + n) continue;
            st4(v + (size_t)(p0 + r + j - base) * stride + (size_t)h * hd + d,
                (f32x4){(int8_t)(w[0] >> (8 * j)) * s, (int8_t)(w[1] >> (8 * j)) * s, (int8_t)(w[2] >> (8 * j)) * s,
                        (int8_t)(w[3] >> (8 * j)) * s}, al);
        }
    }
}

extern "C" hipError_t sgk_kv8_load(const int8_t *codes, const float *scales, float *k, float *v, uint64_t stride,
                                   uint32_t n_kv, uint32_t hd, uint32_t block, uint32_t base, uint32_t n, hipStream_t s) {
    if (!n) return hipSuccess;
    if (!sgk_kv8_shape_ok(n_kv, hd, block) || ((uintptr_t)codes & 15)) return hipErrorInvalidValue;
    const int al = !((uintptr_t)k & 15) && !((uintptr_t)v & 15) && stride % 4 == 0;
    const uint32_t tiles = (uint32_t)(((uint64_t)base + n + KV8_T - 1) / KV8_T) - base / KV8_T;
    hipLaunchKernelGGL(k_kv8_load, dim3(tiles, n_kv, 2), dim3(TPB), 0, s, codes, scales, k, v, stride, n_kv, hd, block, base, n, al);
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Attention of few rows (tokens x the query heads of one kv head, at most 16),
// split over the keys: decode, and chunks of a few tokens. Every wave streams
// its own steps of 32 keys straight from the cache into operands:
//  - q in fixed point against its row's largest element, 24 bits as three int8
//    digits (q = sq (65536 d2 + 256 d1 + d0)): the score product is three
//    v_mfma_i32_16x16x64_i8 on the key codes as they lie, its sums exact, and
//    the keys are never converted;
//  - S^T = K Q^T leaves lane (li, lg) row li's scores of keys 4 lg .. 4 lg + 3
//    of both tiles, the order of the value records' dwords, so V^T P^T runs on
//    v_mfma_f32_16x16x32_f16 with the codes as f16 (exact) and p in two halves;
//  - the values' scale goes into p: w = p s_V. The running maximum is taken
//    over score + log2 s_V, so that w <= 2^12 whatever the scales are, while
//    the sum of p, at most 2^92 a key (log2 s_V >= -80), stays in f32's range.
//    2^12 keeps w's lower half above f16's subnormals down to 2^-26 of the
//    largest.
// No barrier or LDS in the key loop; the waves' maxima, sums and outputs join
// at the end. Bound by the cache's bytes.
// ---------------------------------------------------------------------------
struct kv8_part { float *m, *s, *acc; };    // [token][head][split] maxima and sums, [..][hd] outputs; NULL: one split

#define KV8_P2 12.0f

// 16 f32 of a row as the three digits' operand bytes
__device__ __forceinline__ void q_digits(const float (&x)[16], float inv, v4i &d0, v4i &d1, v4i &d2) {
#pragma unroll
    for (int w = 0; w < 4; w++) {
        uint32_t b0 = 0, b1 = 0, b2 = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int q = (int)rintf(x[4 * w + e] * inv);
            const int l0 = (int8_t)q, r1 = (q - l0) >> 8, l1 = (int8_t)r1, l2 = (r1 - l1) >> 8;
            b0 |= (uint32_t)(l0 & 0xFF) << (8 * e);
            b1 |= (uint32_t)(l1 & 0xFF) << (8 * e);
            b2 |= (uint32_t)(l2 & 0xFF) << (8 * e);
        }
        d0[w] = (int)b0; d1[w] = (int)b1; d2[w] = (int)b2;
    }
}
// A row's q (spread over the four lanes of its column) as digits; returns the
// factor of the integer scores, sq * mul, NaN if an element is not finite.
template <int NC>
__device__ __forceinline__ float q_row(const float *q, bool on, bool al, uint32_t lg, float mul, v4i (&d)[3][NC]) {
    float x[NC][16];
    uint32_t mx = 0;
#pragma unroll
    for (int c = 0; c < NC; c++)
#pragma unroll
        for (int w = 0; w < 4; w++) {
            f32x4 v = {0.f, 0.f, 0.f, 0.f};
            if (on) v = ld4(q + 64 * c + 16 * lg + 4 * w, al);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                x[c][4 * w + e] = v[e];
                mx = max(mx, __float_as_uint(v[e]) & 0x7FFFFFFFu);
            }
        }
    mx = max(mx, swap16(mx));
    mx = max(mx, swap32(mx));
    const bool bad = mx >= 0x7F800000u;
    float am = bad ? 0.0f : __uint_as_float(mx);
    const float up = am < 0x1p-60f ? 0x1p64f : 1.0f;    // a row near the end of the range, times 2^64
    am *= up;
    const float inv = am > 0.0f ? 8323072.0f / am : 0.0f;       // 127 * 65536
#pragma unroll
    for (int c = 0; c < NC; c++) {
#pragma unroll
        for (int e = 0; e < 16; e++) x[c][e] = bad ? 0.0f : x[c][e] * up;
        q_digits(x[c], inv, d[0][c], d[1][c], d[2][c]);
    }
    return bad ? NAN : am / 8323072.0f * mul / up;
}
// the score sums of the three digits as one float (a2 * 256 + a1 < 2^31)
__device__ __forceinline__ float q_join(int a0, int a1, int a2) {
    return fmaf((float)(a2 * 256 + a1), 256.0f, (float)a0);
}
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

// One tile group's scores (UN tiles of 16 keys) to weights, online: updates the
// running maximum and sum of the row, gives the weights' f16 halves in operand
// order and what the output so far is to be multiplied by. MASK: key 16 u +
// 4 lg + e is visible up to rel (keys before the group's first make it
// negative); without it all are.
template <int UN, bool MASK>
__device__ __forceinline__ float softmax_step(float (&sc)[UN][4], const float (&vs)[UN], int rel, float &mrun, float &lsum,
                                              f16x8 (&ph)[UN / 2], f16x8 (&pl)[UN / 2]) {
    const int lg4 = (threadIdx.x & 63) >> 4 << 2;
    float tm = -INFINITY;
#pragma unroll
    for (int u = 0; u < UN; u++) {
        if (MASK) {
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (16 * u + lg4 + e > rel) sc[u][e] = -INFINITY;
        }
        const float m4 = fmaxf(fmaxf(sc[u][0], sc[u][1]), fmaxf(sc[u][2], sc[u][3]));
        tm = fmaxf(tm, m4 + __builtin_amdgcn_logf(fmaxf(vs[u], 0x1p-80f)));
    }
    tm = fmaxf(tm, swap16f(tm));
    tm = fmaxf(tm, swap32f(tm));
    const float mnew = fmaxf(mrun, tm), m0 = mnew - KV8_P2;
    const float al = mrun == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mrun - mnew);
    mrun = mnew;
    float l = lsum * al;
#pragma unroll
    for (int u = 0; u < UN; u++) {
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            // masked keys apart: a row with no key yet has m0 = -inf, and a block's scale may be NaN
            const bool vis = !MASK || 16 * u + lg4 + e <= rel;
            const float p = vis ? __builtin_amdgcn_exp2f(sc[u][e] - m0) : 0.0f;
            l += p;
            w[e] = vis ? p * vs[u] : 0.0f;
        }
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
            const f16x2 h = __builtin_convertvector((f32x2){w[e], w[e + 1]}, f16x2);
            const int at = 4 * (u & 1) + e;
            ph[u / 2][at] = h[0];
            ph[u / 2][at + 1] = h[1];
            pl[u / 2][at] = (_Float16)fmaf((float)h[0], -1.0f, w[e]);
            pl[u / 2][at + 1] = (_Float16)fmaf((float)h[1], -1.0f, w[e + 1]);
        }
    }
    lsum = l;
    return al;
}

template <int HD>
__global__ void __launch_bounds__(TPB, 2) k_kv8_wave(sgk_kv8_attn a, kv8_part part, int al) {
    constexpr int NC = HD / 64, NT = HD / 16, OLD = HD + 4;
    __shared__ float wm[4][16], wl[4][16];
    __shared__ __align__(16) float ob[2][16 * OLD];
    const uint32_t t = threadIdx.x, lane = t & 63, li = lane & 15, lg = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const uint32_t hk = blockIdx.y, sp = blockIdx.x, S = gridDim.x, G = a.n_heads / a.n_kv, R = a.ntok * G;
    const uint32_t ntile = (uint32_t)(((uint64_t)a.base + a.ntok + KV8_T - 1) / KV8_T), nstep = (ntile + 1) / 2;
    const uint32_t s0 = (uint32_t)((uint64_t)sp * nstep / S), s1 = (uint32_t)((uint64_t)(sp + 1) * nstep / S);
    const uint32_t bsh = __builtin_ctz(a.block / KV8_T);
    const uint32_t tok = li < R ? li / G : 0, rpos = a.base + tok;
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
    if (step < s1) {
        load_s(step);
        load_k(step);
        load_v(step);
    }
    v4i qd[3][NC];
    const float qf = q_row<NC>(a.q + tok * a.q_tok + (size_t)(hk * G + li % G) * a.q_stride, li < R, al, lg,
                               a.scale * 1.44269504088896340736f, qd);
    f32x4 o[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) o[n] = (f32x4){0.f, 0.f, 0.f, 0.f};
    float mrun = -INFINITY, lsum = 0.0f;
    for (; step < s1; step += 4) {
        float sc[2][4];
#pragma unroll
        for (int u = 0; u < 2; u++) { ks[u] = nks[u]; vs[u] = nvs[u]; }
#pragma unroll
        for (int u = 0; u < 2; u++) {
            v4i s[3] = {{0, 0, 0, 0}, {0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int d = 0; d < 3; d++)
                    s[d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(v4i, kr[u][c]), qd[d][c], s[d], 0, 0, 0);
            const float f = qf * ks[u];
#pragma unroll
            for (int e = 0; e < 4; e++) sc[u][e] = q_join(s[0][e], s[1][e], s[2][e]) * f;
        }
        const bool more = step + 4 < s1;
        if (more) { load_s(step + 4); load_k(step + 4); }
        f16x8 ph[1], pl[1];
        const float al2 = step * 32 + 31 <= a.base      // every row sees every key
                              ? softmax_step<2, false>(sc, vs, 0, mrun, lsum, ph, pl)
                              : softmax_step<2, true>(sc, vs, (int)(rpos - step * 32), mrun, lsum, ph, pl);
        if (__builtin_amdgcn_ballot_w64(al2 != 1.0f)) {
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
        if (more) load_v(step + 4);
    }
    // join the four waves: maxima and sums first, then outputs 2 + 0, 3 + 1, both
    lsum += swap16f(lsum);
    lsum += swap32f(lsum);
    if (lg == 0) { wm[wave][li] = mrun; wl[wave][li] = lsum; }
    __syncthreads();
    const float M = fmaxf(fmaxf(wm[0][li], wm[1][li]), fmaxf(wm[2][li], wm[3][li]));
    const float f = mrun == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mrun - M);
#pragma unroll
    for (int n = 0; n < NT; n++) o[n] *= f;
    float *mine = &ob[wave & 1][li * OLD + 4 * lg];
    if (wave >= 2) {
#pragma unroll
        for (int n = 0; n < NT; n++) *(f32x4 *)(mine + 16 * n) = o[n];
    }
    __syncthreads();
    if (wave < 2) {
#pragma unroll
        for (int n = 0; n < NT; n++) *(f32x4 *)(mine + 16 * n) += o[n];
    }
    __syncthreads();
    for (uint32_t i = t; i < R * (HD / 4); i += TPB) {
        const uint32_t r = i / (HD / 4), d = i % (HD / 4) * 4;
        const f32x4 v = *(const f32x4 *)&ob[0][r * OLD + d] + *(const f32x4 *)&ob[1][r * OLD + d];
        const float m = fmaxf(fmaxf(wm[0][r], wm[1][r]), fmaxf(wm[2][r], wm[3][r]));
        float l = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; w++)
            l += wl[w][r] * (wm[w][r] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(wm[w][r] - m));
        const size_t row = (size_t)(r / G) * a.n_heads + hk * G + r % G;
        if (S == 1) {
            st4(a.out + row * HD + d, v / l, !((uintptr_t)a.out & 15));
        } else {
            *(f32x4 *)(part.acc + (row * S + sp) * HD + d) = v;
            // base e for the combine; a sum that is NaN has to reach it whatever the maximum
            if (d == 0) { part.m[row * S + sp] = l != l ? 0.0f : m * 0.69314718055994530942f; part.s[row * S + sp] = l; }
        }
    }
}

// ---------------------------------------------------------------------------
// Attention of many rows: a workgroup takes NW x CT x 16 consecutive rows
// (token-major, the query heads of one kv head inside a token, so any group
// size fills them) and walks its keys in tiles of 64, staged once in LDS for
// all of them: the key codes as they lie (1 KB per operand fragment, 16 bytes
// a lane, no bank conflict), the value codes turned into f16 on the way. The
// arithmetic is the wave form's; a wave holds CT column tiles of 16 rows.
// Both tiles are double-buffered: the next tile's loads are requested right
// after a barrier, stored behind the current tile's products, one barrier per
// tile. Grid: (row block, kv head, key split), the longest rows first.
// ---------------------------------------------------------------------------
template <int HD, int NW, int CT>
__global__ void __launch_bounds__(NW * 64) k_kv8_tile(sgk_kv8_attn a, kv8_part part, int al) {
    constexpr int NC = HD / 64, NT = HD / 16, NTH = NW * 64, ROWS = NW * CT * 16;
    constexpr int KCH = 4 * NC * 64, VUN = 2 * NC * 64;     // 16-byte chunks of keys, units (two chunks) of values
    constexpr int KPT = (KCH + NTH - 1) / NTH, VPT = (VUN + NTH - 1) / NTH;
    __shared__ v4u kb[2][KCH];
    __shared__ v4u vb[2][2 * NT * 64];
    const uint32_t t = threadIdx.x, lane = t & 63, li = lane & 15, lg = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const uint32_t hk = blockIdx.y, sp = blockIdx.z, S = gridDim.z, G = a.n_heads / a.n_kv;
    const uint64_t R = (uint64_t)a.ntok * G, r0 = (uint64_t)(gridDim.x - 1 - blockIdx.x) * ROWS;
    const uint32_t lastk = a.base + (uint32_t)(min(r0 + ROWS, R) - 1) / G;      // the block's last visible key
    const uint32_t nrec = lastk / KV8_T + 1, nt = lastk / 64 + 1;
    const uint32_t k0 = (uint32_t)((uint64_t)sp * nt / S), k1 = (uint32_t)((uint64_t)(sp + 1) * nt / S);
    const uint32_t bsh = __builtin_ctz(a.block / KV8_T);
    const size_t rec = (size_t)a.n_kv * (2 * KV8_T * HD);
    const int8_t *codes = a.codes + (size_t)hk * (2 * KV8_T * HD);
    const float *scales = a.scales + 2 * hk;
    const size_t srec = 2 * (size_t)a.n_kv;

    v4u kr[KPT], vr[VPT][2];
    auto load = [&](uint32_t kt) {
#pragma unroll
        for (int x = 0; x < KPT; x++) {
            const uint32_t i = t + x * NTH;
            if (KCH % NTH == 0 || i < KCH)
                kr[x] = *(const v4u *)(codes + min(4 * kt + i / (NC * 64), nrec - 1) * rec + i % (NC * 64) * 16);
        }
#pragma unroll
        for (int x = 0; x < VPT; x++) {
            const uint32_t i = t + x * NTH;
            if (VUN % NTH == 0 || i < VUN)
#pragma unroll
                for (int h = 0; h < 2; h++)
                    vr[x][h] = *(const v4u *)(codes + min(4 * kt + i / (NC * 64) * 2 + h, nrec - 1) * rec + KV8_T * HD +
                                              i % (NC * 64) * 16);
        }
    };
    auto stage = [&](int b) {
#pragma unroll
        for (int x = 0; x < KPT; x++) {
            const uint32_t i = t + x * NTH;
            if (KCH % NTH == 0 || i < KCH) kb[b][i] = kr[x];
        }
#pragma unroll
        for (int x = 0; x < VPT; x++) {
            const uint32_t i = t + x * NTH;
            if (VUN % NTH == 0 || i < VUN)
#pragma unroll
                for (int j = 0; j < 4; j++)         // fragment (pair, dim tile 4 c + j)
                    vb[b][(i / 64 * 4 + j) * 64 + i % 64] = __builtin_bit_cast(v4u, codes_f16(vr[x][0][j], vr[x][1][j]));
        }
    };

    if (k0 < k1) load(k0);
    v4i qd[CT][3][NC];
    float qf[CT], mrun[CT], lsum[CT];
    uint32_t rpos[CT];
    f32x4 o[CT][NT];
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
        const uint64_t r = r0 + (wave * CT + ct) * 16 + li;
        const uint32_t tok = r < R ? (uint32_t)(r / G) : 0, g = r < R ? (uint32_t)(r % G) : 0;
        rpos[ct] = a.base + tok;
        qf[ct] = q_row<NC>(a.q + tok * a.q_tok + (size_t)(hk * G + g) * a.q_stride, r < R, al, lg,
                           a.scale * 1.44269504088896340736f, qd[ct]);
        mrun[ct] = -INFINITY;
        lsum[ct] = 0.0f;
#pragma unroll
        for (int n = 0; n < NT; n++) o[ct][n] = (f32x4){0.f, 0.f, 0.f, 0.f};
    }
    // the wave's first and last visible keys: no mask up to the one, no work past the other
    const uint64_t rw = r0 + wave * CT * 16;
    const bool on = rw < R;
    const uint32_t wfirst = on ? a.base + (uint32_t)(rw / G) : 0, wlast = on ? a.base + (uint32_t)((min(rw + CT * 16, R) - 1) / G) : 0;
    if (k0 < k1) stage(0);
    __syncthreads();
    for (uint32_t kt = k0; kt < k1; kt++) {
        const int b = (kt - k0) & 1;
        const bool more = kt + 1 < k1;
        if (more) load(kt + 1);
        if (on && kt * 64 <= wlast) {
            const bool whole = kt * 64 + 63 <= wfirst;
            float ks[4], vs[4], sc[CT][4][4];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const float *p = scales + (size_t)(min(4 * kt + u, nrec - 1) >> bsh) * srec;
                ks[u] = p[0];
                vs[u] = p[1];
            }
#pragma unroll
            for (int u = 0; u < 4; u++) {
                v4i s[CT][3];
#pragma unroll
                for (int ct = 0; ct < CT; ct++)
#pragma unroll
                    for (int d = 0; d < 3; d++) s[ct][d] = (v4i){0, 0, 0, 0};
#pragma unroll
                for (int c = 0; c < NC; c++) {
                    const v4i kf = __builtin_bit_cast(v4i, kb[b][(u * NC + c) * 64 + lane]);
#pragma unroll
                    for (int ct = 0; ct < CT; ct++)
#pragma unroll
                        for (int d = 0; d < 3; d++)
                            s[ct][d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kf, qd[ct][d][c], s[ct][d], 0, 0, 0);
                }
#pragma unroll
                for (int ct = 0; ct < CT; ct++)
#pragma unroll
                    for (int e = 0; e < 4; e++) sc[ct][u][e] = q_join(s[ct][0][e], s[ct][1][e], s[ct][2][e]) * (qf[ct] * ks[u]);
            }
            f16x8 ph[CT][2], pl[CT][2];
#pragma unroll
            for (int ct = 0; ct < CT; ct++) {
                const float al2 = whole ? softmax_step<4, false>(sc[ct], vs, 0, mrun[ct], lsum[ct], ph[ct], pl[ct])
                                        : softmax_step<4, true>(sc[ct], vs, (int)(rpos[ct] - kt * 64), mrun[ct], lsum[ct], ph[ct], pl[ct]);
                if (__builtin_amdgcn_ballot_w64(al2 != 1.0f)) {
#pragma unroll
                    for (int n = 0; n < NT; n++) o[ct][n] *= al2;
                }
            }
#pragma unroll
            for (int m = 0; m < 2; m++)
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    const f16x8 vf = __builtin_bit_cast(f16x8, vb[b][(m * NT + n) * 64 + lane]);
#pragma unroll
                    for (int ct = 0; ct < CT; ct++) {
                        o[ct][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, ph[ct][m], o[ct][n], 0, 0, 0);
                        o[ct][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pl[ct][m], o[ct][n], 0, 0, 0);
                    }
                }
        }
        if (more) stage(b ^ 1);
        __syncthreads();
    }
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
        lsum[ct] += swap16f(lsum[ct]);
        lsum[ct] += swap32f(lsum[ct]);
        const uint64_t r = r0 + (wave * CT + ct) * 16 + li;
        if (r >= R) continue;
        const float l = lsum[ct];
        const size_t row = (size_t)(r / G) * a.n_heads + hk * G + (uint32_t)(r % G);
        if (S == 1) {
            const bool oal = !((uintptr_t)a.out & 15);
#pragma unroll
            for (int n = 0; n < NT; n++) st4(a.out + row * HD + 16 * n + 4 * lg, o[ct][n] / l, oal);
        } else {
            float *acc = part.acc + (row * S + sp) * HD + 4 * lg;
#pragma unroll
            for (int n = 0; n < NT; n++) *(f32x4 *)(acc + 16 * n) = o[ct][n];
            if (lg == 0) { part.m[row * S + sp] = l != l ? 0.0f : mrun[ct] * 0.69314718055994530942f; part.s[row * S + sp] = l; }
        }
    }
}

// How a call runs. Few rows: the key-split form, in as many splits as give
// every wave a step, up to two workgroups per CU (what is resident). More: row
// blocks, one workgroup per CU at a time, their keys split where that shortens
// the launch: rounds x (a part's tiles + KV8_TAIL for its start and end) tiles
// of KV8_TILE_US, against the partials' way to memory and back.
#define KV8_NW 8
#define KV8_CT 1
#define KV8_ROWS (KV8_NW * KV8_CT * 16u)
#define KV8_TILE_US 2.5         /* at head_dim 256 */
#define KV8_TAIL 3.0
#define KV8_PART_BYTES (256ull << 20)
struct kv8_plan { bool wave; uint32_t splits, blocks; };
static kv8_plan kv8_plan_of(const sgk_kv8_attn *a) {
    const uint64_t G = a->n_heads / a->n_kv, rows = a->ntok * G, keys = (uint64_t)a->base + a->ntok, cus = sgk_device_cus();
    kv8_plan p = {rows <= 16, 1, (uint32_t)((rows + KV8_ROWS - 1) / KV8_ROWS)};
    if (p.wave) {
        uint64_t most = 2 * cus / a->n_kv, want = (keys + 127) / 128;
        if (most > 1024) most = 1024;
        if (most < 1) most = 1;
        p.splits = (uint32_t)(want < most ? want : most);
        return p;
    }
    const uint64_t wgs = (uint64_t)p.blocks * a->n_kv, tiles = (keys + 63) / 64, prow = (uint64_t)a->ntok * a->n_heads * a->hd * 4;
    uint64_t most = wgs < cus ? 2 * cus / wgs : 8;
    if (most > 1024) most = 1024;
    if (most > tiles) most = tiles;
    double best = 0.0;
    for (uint64_t S = 1; S <= most && (S == 1 || S * prow <= KV8_PART_BYTES); S++) {
        const double rounds = (double)((wgs * S + cus - 1) / cus), part = (double)((tiles + S - 1) / S) + KV8_TAIL;
        const double cost = rounds * part * KV8_TILE_US * a->hd / 256 + (S > 1 ? 5.0 + (double)(2 * S * prow) / 4.0e6 : 0.0);
        if (S == 1 || cost < best) { best = cost; p.splits = (uint32_t)S; }
    }
    return p;
}

extern "C" uint64_t sgk_kv8_attn_scratch(const sgk_kv8_attn *a) {
    const kv8_plan p = kv8_plan_of(a);
    return p.splits > 1 ? (uint64_t)a->ntok * a->n_heads * p.splits * (a->hd + 2) * 4 : 0;
}

extern "C" hipError_t sgk_kv8_attention(const sgk_kv8_attn *a, void *scratch, hipStream_t s) {
    if (!a->ntok || !a->n_heads) return hipSuccess;
    if (!sgk_kv8_shape_ok(a->n_kv, a->hd, a->block) || ((uintptr_t)a->codes & 15) || a->n_heads % a->n_kv ||
        a->n_heads / a->n_kv > SGK_KV8_MAX_GROUP) return hipErrorInvalidValue;
    const kv8_plan p = kv8_plan_of(a);
    if (p.splits > 1 && !scratch) return hipErrorInvalidValue;
    const int al = !((uintptr_t)a->q & 15) && a->q_stride % 4 == 0 && a->q_tok % 4 == 0;
    const uint64_t rows = (uint64_t)a->ntok * a->n_heads * p.splits;
    kv8_part part = {};
    if (p.splits > 1) {                 // outputs first, as they are stored 16 bytes at a time
        part.acc = (float *)scratch;
        part.m = part.acc + rows * a->hd;
        part.s = part.m + rows;
    }
#define KC(H)                                                                                                                 \
    do {                                                                                                                      \
        if (p.wave) hipLaunchKernelGGL(k_kv8_wave<H>, dim3(p.splits, a->n_kv), dim3(TPB), 0, s, *a, part, al);                \
        else hipLaunchKernelGGL((k_kv8_tile<H, KV8_NW, KV8_CT>), dim3(p.blocks, a->n_kv, p.splits), dim3(KV8_NW * 64), 0, s,  \
                                *a, part, al);                                                                                \
    } while (0)
    switch (a->hd) {
    case 64: KC(64); break;
    case 128: KC(128); break;
    default: KC(256); break;
    }
#undef KC
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.splits == 1) return e;
    sgk_attn c = {};
    c.m = part.m; c.s = part.s; c.acc = part.acc; c.out = a->out; c.n_heads = a->n_heads; c.n_kv = a->n_kv; c.hd = a->hd;
    c.out_tok = a->n_heads * a->hd; c.n_splits = p.splits; c.max_splits = p.splits; c.ntok = a->ntok;
    return sgk_attn_combine(&c, s);
}
