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

extern "C" hipError_t sgk_kv8_attention(const sgk_kv8_attn *a, hipStream_t s) {
    if (!a->ntok || !a->n_heads) return hipSuccess;
    if (!sgk_kv8_shape_ok(a->n_kv, a->hd, a->block) || ((uintptr_t)a->codes & 15)) return hipErrorInvalidValue;
    for (uint32_t z = 0; z < a->ntok; z += 32768) {
        sgk_kv8_attn b = *a;
        b.q += z * a->q_tok; b.out += (size_t)z * a->n_heads * a->hd; b.base += z;
        b.ntok = a->ntok - z < 32768 ? a->ntok - z : 32768;
        hipLaunchKernelGGL(k_kv8_attn, dim3(a->n_heads, b.ntok), dim3(TPB), 0, s, b);
    }
    return hipGetLastError();
}
