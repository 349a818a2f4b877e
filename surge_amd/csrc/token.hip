// token.hip - the operators on both sides of the layers: rotary positions with
// several axes before attention, and logits under penalties, a bias and a mask
// with the token they choose after the head. Launchers are declared in
// kernels.h; their host checks are in hip.c.
#include "devutil.h"
#include "kernels.h"

// ---------------------------------------------------------------------------
// Rotary positions with three axes. A workgroup takes RA_TOK tokens: first
// their cos and sin per pair, one thread each (the angle and its functions in
// double: a far position times a frequency loses the angle in 32 bits), then
// every head's slice, four dims and their four partners per thread (or the
// dims behind rope_dim, copied). Each element is read and written by one
// thread, both halves of a pair by the same one, so out may be x.
// ---------------------------------------------------------------------------
#define RA_TOK 4u
struct rope_tab { double inv[SGK_ROPE_HALF]; uint8_t axis[SGK_ROPE_HALF]; };

// one slice unit: V dims at d and, below rope_dim, their partners at d + half
template <int V>
__device__ __forceinline__ void rope_unit(const float *x, float *o, uint32_t d, uint32_t half, uint32_t rope_dim, bool copy,
                                          const float *cs) {
    if (d < half) {
        float a[V], b[V];
#pragma unroll
        for (int e = 0; e < V; e++) { a[e] = x[d + e]; b[e] = x[d + half + e]; }
#pragma unroll
        for (int e = 0; e < V; e++) {
            const float c = cs[d + e], s = cs[half + d + e];
            o[d + e] = a[e] * c - b[e] * s;
            o[d + half + e] = b[e] * c + a[e] * s;
        }
    } else if (copy) {
        const uint32_t t = d - half + rope_dim;     // units past the pairs: the dims behind rope_dim
#pragma unroll
        for (int e = 0; e < V; e++) o[t + e] = x[t + e];
    }
}

template <int V>
__global__ void __launch_bounds__(TPB) k_rope_axes(sgk_rope_axes_args a, rope_tab tab) {
    __shared__ float cs[RA_TOK][2 * SGK_ROPE_HALF];
    const uint32_t half = a.rope_dim / 2, t = threadIdx.x;
    // a slice's units: half / V of pairs, then (head_dim - rope_dim) / V copies
    const uint32_t upr = (a.head_dim - half) / V;
    const bool copy = a.x != a.out;
    for (uint64_t z0 = (uint64_t)blockIdx.x * RA_TOK; z0 < a.n; z0 += (uint64_t)gridDim.x * RA_TOK) {
        const uint32_t nt = min((uint64_t)RA_TOK, a.n - z0);
        __syncthreads();
        for (uint32_t i = t; i < nt * half; i += TPB) {
            const uint32_t z = i / half, f = i % half;
            double s, c;
            sincos((double)a.pos[(uint64_t)tab.axis[f] * a.n + z0 + z] * tab.inv[f], &s, &c);
            cs[z][f] = (float)c;
            cs[z][half + f] = (float)s;
        }
        __syncthreads();
        const uint32_t per = a.heads * upr;
        for (uint32_t i = t; i < nt * per; i += TPB) {
            const uint32_t z = i / per, h = (i % per) / upr, u = i % upr;
            const uint64_t at = (z0 + z) * a.row + (uint64_t)h * a.stride;
            rope_unit<V>(a.x + at, a.out + at, u * V, half, a.rope_dim, copy, cs[z]);
        }
    }
}

extern "C" hipError_t sgk_rope_axes(const sgk_rope_axes_args *a, const double *inv, const uint8_t *axis, hipStream_t s) {
    const uint32_t half = a->rope_dim / 2;
    if (!a->n || !a->heads) return hipSuccess;
    if (!half || half > SGK_ROPE_HALF || a->rope_dim > a->head_dim) return hipErrorInvalidValue;
    rope_tab tab = {};
    for (uint32_t i = 0; i < half; i++) { tab.inv[i] = inv[i]; tab.axis[i] = axis[i]; }
    const uint64_t blocks = ((uint64_t)a->n + RA_TOK - 1) / RA_TOK;
    const uint32_t grid = (uint32_t)(blocks < 65536 ? blocks : 65536);
    hipLaunchKernelGGL(k_rope_axes<1>, dim3(grid), dim3(TPB), 0, s, *a, tab);
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Token counts: integer atomics, so the order of equal ids does not matter.
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(TPB) k_zero_u32(uint32_t *p, uint64_t n) {
    for (uint64_t i = (uint64_t)blockIdx.x * TPB + threadIdx.x; i < n; i += (uint64_t)gridDim.x * TPB) p[i] = 0;
}
__global__ void __launch_bounds__(TPB) k_token_counts(const int32_t *ids, uint32_t *counts, uint32_t n, uint32_t vocab,
                                                      uint32_t rows) {
    for (uint32_t r = blockIdx.y; r < rows; r += gridDim.y)
        for (uint64_t i = (uint64_t)blockIdx.x * TPB + threadIdx.x; i < n; i += (uint64_t)gridDim.x * TPB) {
            const uint32_t id = (uint32_t)ids[(uint64_t)r * n + i];
            if (id < vocab) atomicAdd(counts + (uint64_t)r * vocab + id, 1u);
        }
}

extern "C" hipError_t sgk_token_counts(const int32_t *ids, uint32_t *counts, uint32_t n, uint32_t vocab, uint32_t rows,
                                       int clear, hipStream_t s) {
    if (!vocab || !rows) return hipSuccess;
    if (clear) {
        const uint64_t b = ((uint64_t)rows * vocab + TPB - 1) / TPB;
        hipLaunchKernelGGL(k_zero_u32, dim3((uint32_t)(b < 2048 ? b : 2048)), dim3(TPB), 0, s, counts, (uint64_t)rows * vocab);
    }
    if (n) {
        const uint64_t b = ((uint64_t)n + TPB - 1) / TPB;
        hipLaunchKernelGGL(k_token_counts, dim3((uint32_t)(b < 1024 ? b : 1024), rows < 65535 ? rows : 65535), dim3(TPB), 0, s,
                           ids, counts, n, vocab, rows);
    }
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Logits. Workgroups (part, row) write the row's processed logits and each its
// best (value, id); a second launch folds the parts. The best is the largest
// value, ties to the lowest id, so no order of the folds changes it. NaN is
// never better, and -inf neither: a row with nothing allowed has no token.
// ---------------------------------------------------------------------------
#define LG_PARTS 64u
struct lg_best { float v; uint32_t i; };
#define LG_NONE 0xFFFFFFFFu

__device__ __forceinline__ void lg_better(lg_best &b, float v, uint32_t i) {
    if (v > b.v || (v == b.v && i < b.i && b.i != LG_NONE)) { b.v = v; b.i = i; }
}
__device__ __forceinline__ lg_best lg_fold(lg_best b, lg_best *red) {
    const uint32_t t = threadIdx.x;
    red[t] = b;
    __syncthreads();
    for (uint32_t o = TPB / 2; o; o >>= 1) {
        if (t < o) { lg_best x = red[t]; lg_better(x, red[t + o].v, red[t + o].i); red[t] = x; }
        __syncthreads();
    }
    return red[0];
}
__device__ __forceinline__ float lg_value(const sgk_logits_args &a, float x, uint32_t c, float bias, bool ok) {
    if (c) {
        x = x > 0.0f ? x / a.rep : x * a.rep;
        x = x - (float)c * a.freq - a.pres;
    }
    return ok ? x + bias : -INFINITY;
}

__global__ void __launch_bounds__(TPB) k_logits(sgk_logits_args a, lg_best *part) {
    __shared__ lg_best red[TPB];
    const uint64_t r = blockIdx.y, row = r * a.vocab, words = (a.vocab + 31) / 32;
    lg_best b = {-INFINITY, LG_NONE};
    for (uint64_t i = (uint64_t)blockIdx.x * TPB + threadIdx.x; i < a.vocab; i += (uint64_t)gridDim.x * TPB) {
        const uint32_t c = a.counts ? a.counts[row + i] : 0;
        const bool ok = !a.mask || (a.mask[r * words + i / 32] >> (i % 32) & 1);
        const float x = lg_value(a, a.x[row + i], c, a.bias ? a.bias[i] : 0.0f, ok);
        a.out[row + i] = x;
        lg_better(b, x, (uint32_t)i);
    }
    b = lg_fold(b, red);
    if (threadIdx.x == 0) part[r * gridDim.x + blockIdx.x] = b;
}
__global__ void __launch_bounds__(TPB) k_logits_token(const lg_best *part, uint32_t parts, uint32_t *token) {
    __shared__ lg_best red[TPB];
    lg_best b = {-INFINITY, LG_NONE};
    if (threadIdx.x < parts) b = part[(uint64_t)blockIdx.x * parts + threadIdx.x];
    b = lg_fold(b, red);
    if (threadIdx.x == 0) token[blockIdx.x] = b.i;
}

extern "C" uint64_t sgk_logits_part_bytes(uint32_t rows) { return (uint64_t)rows * LG_PARTS * sizeof(lg_best); }
extern "C" hipError_t sgk_logits(const sgk_logits_args *a, void *part, hipStream_t s) {
    if (!a->vocab || !a->rows) return hipSuccess;
    const uint32_t need = (uint32_t)(((uint64_t)a->vocab + TPB - 1) / TPB), parts = need < LG_PARTS ? need : LG_PARTS;
    hipLaunchKernelGGL(k_logits, dim3(parts, a->rows), dim3(TPB), 0, s, *a, (lg_best *)part);
    hipLaunchKernelGGL(k_logits_token, dim3(a->rows), dim3(TPB), 0, s, (const lg_best *)part, parts, a->token);
    return hipGetLastError();
}
