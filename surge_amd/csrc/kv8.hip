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
    float s = fmaxf(__uint_as_float(poison ? 0 : mx) / 127.0f, poison ? 0.0f : was);
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
// Attention, one workgroup per (token, query head): per tile of 16 positions
// thread (chunk c, position r) sums hd/16 products, 16 chunks per position are
// added through LDS, then thread d accumulates dim d. The running maximum and
// sum are kept per thread, the same in all of them.
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(TPB) k_kv8_attn(sgk_kv8_attn a) {
    __shared__ float qs[256];
    __shared__ float ds[16][KV8_T + 1];
    const uint32_t t = threadIdx.x, h = blockIdx.x, z = blockIdx.y, hd = a.hd, hk = h / (a.n_heads / a.n_kv);
    const uint32_t last = a.base + z;
    const float *q = a.q + z * a.q_tok + (size_t)h * a.q_stride;
    if (t < hd) qs[t] = q[t];
    __syncthreads();
    const uint32_t c = t / 16, r = t % 16, cw = hd / 16;
    float m = -INFINITY, l = 0.0f, o = 0.0f;
    for (uint32_t tile = 0; tile <= last / KV8_T; tile++) {
        const float *sc = a.scales + ((size_t)(tile * KV8_T / a.block) * a.n_kv + hk) * 2;
        const int8_t *rec = a.codes + rec_at(tile, a.n_kv, hk, hd);
        float dot = 0.0f;
        for (uint32_t e = 0; e < cw; e++) dot = fmaf(qs[c * cw + e], (float)rec[key_at(r, c * cw + e)], dot);
        ds[c][r] = dot;
        __syncthreads();
        float sv[KV8_T], tm = -INFINITY;
        for (uint32_t j = 0; j < KV8_T; j++) {
            float x = 0.0f;
            for (uint32_t i = 0; i < 16; i++) x += ds[i][j];
            sv[j] = tile * KV8_T + j <= last ? x * sc[0] * a.scale : -INFINITY;
            tm = fmaxf(tm, sv[j]);
        }
        const float mn = fmaxf(m, tm), al = m == -INFINITY ? 0.0f : expf(m - mn);
        m = mn;
        l *= al;
        o *= al;
        for (uint32_t j = 0; j < KV8_T; j++) {
            if (tile * KV8_T + j > last) break;
            const float p = expf(sv[j] - m);
            l += p;
            if (t < hd) o = fmaf(p, (float)rec[KV8_T * hd + val_at(j, t)] * sc[1], o);
        }
        __syncthreads();
    }
    if (t < hd) a.out[((size_t)z * a.n_heads + h) * hd + t] = o / l;
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
        float sc[2][4], tm = -INFINITY;
        const bool whole = step * 32 + 31 <= a.base;            // every row sees every key
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
            const float f = qf * ks[u], lv = __builtin_amdgcn_logf(fmaxf(vs[u], 0x1p-80f));
#pragma unroll
            for (int e = 0; e < 4; e++) {
                sc[u][e] = q_join(s[0][e], s[1][e], s[2][e]) * f;
                if (whole || step * 32 + u * 16 + 4 * lg + e <= rpos) tm = fmaxf(tm, sc[u][e] + lv);
            }
        }
        const bool more = step + 4 < s1;
        if (more) { load_s(step + 4); load_k(step + 4); }
        tm = fmaxf(tm, swap16f(tm));
        tm = fmaxf(tm, swap32f(tm));
        const float mnew = fmaxf(mrun, tm), m0 = mnew - KV8_P2;
        const float al2 = mrun == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mrun - mnew);
        mrun = mnew;
        lsum *= al2;
        f16x8 ph, pl;
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const bool on = whole || step * 32 + u * 16 + 4 * lg + e <= rpos;
                const float p = on ? __builtin_amdgcn_exp2f(sc[u][e] - m0) : 0.0f;
                lsum += p;
                const float w = on ? p * vs[u] : 0.0f;
                const _Float16 h = (_Float16)w;
                ph[4 * u + e] = h;
                pl[4 * u + e] = (_Float16)(w - (float)h);
            }
        if (__builtin_amdgcn_ballot_w64(al2 != 1.0f)) {
#pragma unroll
            for (int n = 0; n < NT; n++) o[n] *= al2;
        }
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const f16x8 v = codes_f16(vr[0][c][j], vr[1][c][j]);
                o[4 * c + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, ph, o[4 * c + j], 0, 0, 0);
                o[4 * c + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pl, o[4 * c + j], 0, 0, 0);
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

// How a call runs. Few rows: the key-split form, in as many splits as give
// every wave a step, up to two workgroups per CU (what is resident).
struct kv8_plan { bool wave; uint32_t splits; };
static kv8_plan kv8_plan_of(const sgk_kv8_attn *a) {
    kv8_plan p = {(uint64_t)a->ntok * (a->n_heads / a->n_kv) <= 16, 1};
    const uint64_t steps = ((uint64_t)a->base + a->ntok + 31) / 32;
    if (p.wave) {
        uint64_t most = 2ull * sgk_device_cus() / a->n_kv, want = (steps + 3) / 4;
        if (most > 1024) most = 1024;
        if (most < 1) most = 1;
        p.splits = (uint32_t)(want < most ? want : most);
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
    if (p.wave) {
        const dim3 grid(p.splits, a->n_kv);
        switch (a->hd) {
        case 64: hipLaunchKernelGGL(k_kv8_wave<64>, grid, dim3(TPB), 0, s, *a, part, al); break;
        case 128: hipLaunchKernelGGL(k_kv8_wave<128>, grid, dim3(TPB), 0, s, *a, part, al); break;
        default: hipLaunchKernelGGL(k_kv8_wave<256>, grid, dim3(TPB), 0, s, *a, part, al); break;
        }
        if (p.splits == 1) return hipGetLastError();
        sgk_attn c = {};
        c.m = part.m; c.s = part.s; c.acc = part.acc; c.out = a->out; c.n_heads = a->n_heads; c.n_kv = a->n_kv; c.hd = a->hd;
        c.out_tok = a->n_heads * a->hd; c.n_splits = p.splits; c.max_splits = p.splits; c.ntok = a->ntok;
        const hipError_t e = hipGetLastError();
        return e == hipSuccess ? sgk_attn_combine(&c, s) : e;
    }
    for (uint32_t z = 0; z < a->ntok; z += 32768) {
        sgk_kv8_attn b = *a;
        b.q += z * a->q_tok; b.out += (size_t)z * a->n_heads * a->hd; b.base += z;
        b.ntok = a->ntok - z < 32768 ? a->ntok - z : 32768;
        hipLaunchKernelGGL(k_kv8_attn, dim3(a->n_heads, b.ntok), dim3(TPB), 0, s, b);
    }
    return hipGetLastError();
}
