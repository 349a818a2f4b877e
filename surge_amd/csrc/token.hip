// token.hip - the operators on both sides of the layers: rotary positions with
// several axes before attention, and logits under penalties, a bias and a mask
// with the token they choose after the head. Launchers are declared in
// kernels.h; their host checks are in hip.c.
#include "devutil.h"
#include "kernels.h"

// ---------------------------------------------------------------------------
// Rotary positions with three axes. A workgroup takes a token and some of its
// heads: cos and sin of the token's pairs once, one thread each (the angle and
// its functions in double: a far position times a frequency loses the angle in
// 32 bits), then a slice (token, head) per 2^wl lanes. The first slice's loads
// go out before the angles, whose chain is as long as a trip to memory.
// Bound by memory for many tokens (4093 x 24 heads of 256, 201 MB: 43 us, a copy
// of them 39), by that chain for one (3.0 us).
// ---------------------------------------------------------------------------
// The frequencies are exp2 of a product here (0.35 us less for one token than a
// table among the arguments, which lie in the host's memory).
__device__ __forceinline__ void rope_angles(const sgk_rope_axes_args &a, uint64_t z, float *cs) {
    const uint32_t half = a.rope_dim / 2, t = threadIdx.x;
    __syncthreads();
    if (t < half) {
        const uint32_t m = t % 3, turns = m == 1 ? a.sections[1] : a.sections[2];
        const uint32_t axis = a.order ? (m && t < 3 * turns ? m : 0) : t < a.sections[0] ? 0 : t < a.sections[0] + a.sections[1] ? 1 : 2;
        double s, c;
        sincos((double)a.pos[(uint64_t)axis * a.n + z] * exp2((double)t * a.step), &s, &c);
        cs[t] = (float)c;
        cs[half + t] = (float)s;
    }
    __syncthreads();
}

// Four dims per lane, the whole slice in one 16-byte load and store of a lane
// group, the partners' dims in a second load (from cache). A group reads all of
// a slice before it writes, so out may be x. hper: heads per workgroup.
__global__ void __launch_bounds__(TPB) k_rope_axes4(sgk_rope_axes_args a, uint32_t hper, uint32_t wl) {
    __shared__ __align__(16) float cs[2 * SGK_ROPE_HALF];
    const uint32_t half = a.rope_dim / 2, t = threadIdx.x, d = (t & ((1u << wl) - 1)) * 4, hstep = TPB >> wl;
    const uint32_t h0 = blockIdx.y * hper, h1 = min(h0 + hper, a.heads);
    const bool on = d < a.head_dim, first = d < half, turn = d < a.rope_dim;
    const uint32_t w = first ? d : d - half;
    for (uint64_t z = blockIdx.x; z < a.n; z += gridDim.x) {
        uint32_t h = h0 + (t >> wl);
        f32x4 v, o;
        uint64_t at;
        auto fetch = [&]() {
            at = z * a.row + (uint64_t)h * a.stride + d;
            if (h < h1 && on) {
                v = *(const f32x4 *)(a.x + at);
                if (turn) o = *(const f32x4 *)(first ? a.x + at + half : a.x + at - half);
            }
        };
        fetch();
        rope_angles(a, z, cs);
        f32x4 c, s;
        if (turn) {
            c = *(const f32x4 *)&cs[w];
            s = *(const f32x4 *)&cs[half + w];
            if (first) s = -s;
        }
        while (h < h1) {
            if (on) *(f32x4 *)(a.out + at) = turn ? v * c + o * s : v;
            h += hstep;
            fetch();
        }
    }
}

// Any size and alignment: a lane takes a pair, or a dim behind rope_dim.
__global__ void __launch_bounds__(TPB) k_rope_axes1(sgk_rope_axes_args a, uint32_t hper, uint32_t wl) {
    __shared__ float cs[2 * SGK_ROPE_HALF];
    const uint32_t half = a.rope_dim / 2, t = threadIdx.x, units = a.head_dim - half;
    const uint32_t h0 = blockIdx.y * hper, h1 = min(h0 + hper, a.heads);
    for (uint64_t z = blockIdx.x; z < a.n; z += gridDim.x) {
        rope_angles(a, z, cs);
        for (uint32_t h = h0 + (t >> wl); h < h1; h += TPB >> wl)
            for (uint32_t u = t & ((1u << wl) - 1); u < units; u += 1u << wl) {
                const uint64_t at = z * a.row + (uint64_t)h * a.stride + u;
                if (u < half) {
                    const float lo = a.x[at], hi = a.x[at + half], c = cs[u], s = cs[half + u];
                    a.out[at] = lo * c - hi * s;
                    a.out[at + half] = hi * c + lo * s;
                } else {
                    a.out[at + half] = a.x[at + half];
                }
            }
    }
}

extern "C" hipError_t sgk_rope_axes(const sgk_rope_axes_args *a, hipStream_t s, hipEvent_t done) {
    const uint32_t half = a->rope_dim / 2;
    if (!a->n || !a->heads) return hipSuccess;
    if (!half || half > SGK_ROPE_HALF || a->rope_dim > a->head_dim || a->head_dim > 256) return hipErrorInvalidValue;
    const bool v4 = !(((uintptr_t)a->x | (uintptr_t)a->out) & 15) && a->row % 4 == 0 && a->stride % 4 == 0 && half % 4 == 0 &&
                    a->head_dim % 4 == 0;
    const uint32_t units = v4 ? a->head_dim / 4 : a->head_dim - half;
    uint32_t wl = 0;
    while (wl < 6 && (1u << wl) < units) wl++;
    // few tokens: their heads spread until every CU has a workgroup, a slice to a lane group
    const uint32_t per = TPB >> wl, want = (uint32_t)(((uint64_t)sgk_device_cus() + a->n - 1) / a->n);
    const uint32_t hs = min(want, (a->heads + per - 1) / per), hper = (a->heads + hs - 1) / hs;
    const dim3 grid(min(a->n, 1u << 20), (a->heads + hper - 1) / hper);
    if (v4) launch(k_rope_axes4, grid, TPB, s, done, *a, hper, wl);
    else launch(k_rope_axes1, grid, TPB, s, done, *a, hper, wl);
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Token counts. Text repeats itself: added one by one, the commonest id's
// additions to one address wait for each other across the chip (about 30 ns
// each; 16 rows of 32000 ids with a fifth of them alike took 182 us). So a
// workgroup first counts TC_IDS ids in a table in LDS, open addressing, then
// adds each distinct id once. Integer additions: their order does not matter.
// ---------------------------------------------------------------------------
#define TC_IDS 2048u
#define TC_SLOTS 4096u      // twice the ids, so a free slot is always found
#define TC_FREE 0xFFFFFFFFu
__global__ void __launch_bounds__(TPB) k_zero_u32(uint32_t *p, uint64_t n) {
    for (uint64_t i = (uint64_t)blockIdx.x * TPB + threadIdx.x; i < n; i += (uint64_t)gridDim.x * TPB) p[i] = 0;
}
__global__ void __launch_bounds__(TPB) k_token_counts(const int32_t *ids, uint32_t *counts, uint32_t n, uint32_t vocab,
                                                      uint32_t rows) {
    __shared__ uint32_t key[TC_SLOTS], num[TC_SLOTS];
    const uint32_t t = threadIdx.x;
    for (uint32_t r = blockIdx.y; r < rows; r += gridDim.y)
        for (uint64_t i0 = (uint64_t)blockIdx.x * TC_IDS; i0 < n; i0 += (uint64_t)gridDim.x * TC_IDS) {
            const uint32_t m = (uint32_t)min((uint64_t)TC_IDS, n - i0);
            uint32_t id[TC_IDS / TPB];
#pragma unroll
            for (uint32_t x = 0; x < TC_IDS / TPB; x++) {
                const uint32_t i = t + x * TPB;
                id[x] = i < m ? (uint32_t)ids[(uint64_t)r * n + i0 + i] : TC_FREE;
            }
            for (uint32_t i = t; i < TC_SLOTS; i += TPB) { key[i] = TC_FREE; num[i] = 0; }
            __syncthreads();
#pragma unroll
            for (uint32_t x = 0; x < TC_IDS / TPB; x++) {
                if (id[x] >= vocab) continue;
                for (uint32_t s = id[x] * 2654435761u >> 20;; s = (s + 1) & (TC_SLOTS - 1)) {
                    const uint32_t was = atomicCAS(&key[s], TC_FREE, id[x]);
                    if (was != TC_FREE && was != id[x]) continue;
                    atomicAdd(&num[s], 1u);
                    break;
                }
            }
            __syncthreads();
            for (uint32_t i = t; i < TC_SLOTS; i += TPB)
                if (key[i] != TC_FREE) atomicAdd(counts + (uint64_t)r * vocab + key[i], num[i]);
            __syncthreads();
        }
}

// Up to TR_MOST ids a row: a workgroup owns TR_IDS ids of the vocabulary (TR_FEW
// where those still find a CU each: 900 ids of 1 row 10.8 us a call against 11.3,
// of 16 rows 15.2 against 13.0), reads the row's whole history and counts its own
// in LDS, alike neighbours of a thread at once, so nothing is cleared first and no
// two additions meet in memory. Whole call, us, 151936 ids, cleared, this form /
// the table form, for Zipf's law with exponent 1.2 and for one id only: 900 ids of
// 1 row 10.9 / 16.6, 11.3 / 16.7; 32000 of 1 row 15.6 / 21.2, 14.1 / 20.8; 131072 of
// 16 rows 41 / 103, 29 / 33; 262144 of 1 row 52 / 54, 47 / 21. Past TR_MOST the walk
// over the history decides, and the table form spreads that.
#define TR_IDS 8192u
#define TR_FEW 2048u
#define TR_THREADS 1024
#define TR_U 8u
#define TR_MOST 131072u
__global__ void __launch_bounds__(TR_THREADS) k_token_recount(const int32_t *ids, uint32_t *counts, uint32_t n, uint32_t vocab, uint32_t range,
                                                              int clear) {
    __shared__ uint32_t num[TR_IDS];
    const uint32_t t = threadIdx.x, v0 = blockIdx.x * range, nv = min(range, vocab - v0);
    const uint32_t r = blockIdx.y;
    for (uint32_t i = t; i < nv; i += TR_THREADS) num[i] = 0;
    __syncthreads();
    const int32_t *row = ids + (uint64_t)r * n;
    constexpr uint32_t U = TR_U;
    for (uint32_t i0 = 0; i0 < n; i0 += U * TR_THREADS) {
        uint32_t id[U];
#pragma unroll
        for (uint32_t x = 0; x < U; x++) {
            const uint32_t i = i0 + x * TR_THREADS + t;
            id[x] = i < n ? (uint32_t)row[i] : 0xFFFFFFFFu;
        }
        uint32_t c = 1;         // of id[x] so far: alike neighbours are added once
#pragma unroll
        for (uint32_t x = 0; x < U; x++) {
            if (x + 1 < U && id[x] == id[x + 1]) { c++; continue; }
            if (id[x] - v0 < nv) atomicAdd(&num[id[x] - v0], c);
            c = 1;
        }
    }
    __syncthreads();
    uint32_t *out = counts + (uint64_t)r * vocab + v0;
    for (uint32_t i = t; i < nv; i += TR_THREADS) {
        if (clear) out[i] = num[i];
        else if (num[i]) out[i] += num[i];
    }
}

extern "C" hipError_t sgk_token_counts(const int32_t *ids, uint32_t *counts, uint32_t n, uint32_t vocab, uint32_t rows,
                                       int clear, hipStream_t s, hipEvent_t done) {
    if (!vocab || !rows || (!n && !clear)) return hipErrorInvalidValue;     // nothing to launch, nothing to wait for
    if (n && n <= TR_MOST) {
        const uint32_t few = (vocab + TR_FEW - 1) / TR_FEW, range = (uint64_t)few * rows <= sgk_device_cus() ? TR_FEW : TR_IDS;
        launch(k_token_recount, dim3((vocab + range - 1) / range, rows), TR_THREADS, s, done, ids, counts, n, vocab, range, clear);
        return hipGetLastError();
    }
    if (clear) {
        const uint64_t b = ((uint64_t)rows * vocab + TPB - 1) / TPB;
        launch(k_zero_u32, dim3((uint32_t)(b < 2048 ? b : 2048)), TPB, s, n ? NULL : done, counts, (uint64_t)rows * vocab);
    }
    if (n) {
        const uint64_t b = ((uint64_t)n + TC_IDS - 1) / TC_IDS;
        launch(k_token_counts, dim3((uint32_t)(b < 1024 ? b : 1024), rows), TPB, s, done, ids, counts, n, vocab, rows);
    }
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Logits. Workgroups (part, row) write the row's processed logits and each its
// best (value, id); a second launch folds the parts. The best is the largest
// value, ties to the lowest id, so no order of the folds changes it. NaN is
// never better, and -inf neither: a row with nothing allowed has no token.
// A thread takes four neighbouring ids a step, 16 bytes of each input where
// addresses allow. Bound by the latency of its two launches: 151936 ids, 1 row
// 4.2 + 2.6 us; 16 rows (29 MB) 9.4 + 2.5-4.
// ---------------------------------------------------------------------------
#define LG_WGS 3200u         // workgroups of all rows together, at most; a row has at least one
struct lg_best { float v; uint32_t i; };
#define LG_NONE 0xFFFFFFFFu

__device__ __forceinline__ void lg_better(lg_best &b, float v, uint32_t i) {
    if (v > b.v || (v == b.v && i < b.i && b.i != LG_NONE)) { b.v = v; b.i = i; }
}
// the best of the workgroup, in thread 0
__device__ __forceinline__ lg_best lg_fold(lg_best b) {
    __shared__ lg_best red[TPB / 64];
#define LG_STEP(F) lg_better(b, __uint_as_float(F(__float_as_uint(b.v))), F(b.i))
    // a partner's NONE is never better: its value is -inf
    LG_STEP(dppu<0xB1>); LG_STEP(dppu<0x4E>); LG_STEP(dppu<0x141>); LG_STEP(dppu<0x128>); LG_STEP(swap16); LG_STEP(swap32);
#undef LG_STEP
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = b;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < TPB / 64; w++) lg_better(b, red[w].v, red[w].i);
    return b;
}
__device__ __forceinline__ float lg_value(const sgk_logits_args &a, float x, uint32_t c, float bias, bool ok) {
    if (c) {
        x = x > 0.0f ? x / a.rep : x * a.rep;
        x = x - (float)c * a.freq - a.pres;
    }
    return ok ? x + bias : -INFINITY;
}

template <bool V4>
__global__ void __launch_bounds__(TPB) k_logits(sgk_logits_args a, lg_best *part) {
    const uint64_t r = blockIdx.y, row = r * a.vocab;
    const uint32_t words = (a.vocab + 31) / 32, quads = (a.vocab + 3) / 4;
    lg_best b = {-INFINITY, LG_NONE};
    for (uint32_t q = blockIdx.x * TPB + threadIdx.x; q < quads; q += gridDim.x * TPB) {
        const uint32_t i = 4 * q, n = V4 ? 4 : min(4u, a.vocab - i);
        float x[4] = {0, 0, 0, 0}, bias[4] = {0, 0, 0, 0};
        uint32_t c[4] = {0, 0, 0, 0};
        const uint32_t bits = a.mask ? a.mask[r * words + i / 32] >> (i % 32) : 0xF;   // four ids share a word
        if (V4) {
            const f32x4 v = *(const f32x4 *)(a.x + row + i);
            const v4u cv = a.counts ? *(const v4u *)(a.counts + row + i) : (v4u){0, 0, 0, 0};
            const f32x4 bv = a.bias ? *(const f32x4 *)(a.bias + i) : (f32x4){0, 0, 0, 0};
#pragma unroll
            for (int e = 0; e < 4; e++) { x[e] = v[e]; c[e] = cv[e]; bias[e] = bv[e]; }
        } else {
#pragma unroll
            for (uint32_t e = 0; e < 4; e++) {
                if (e >= n) break;
                x[e] = a.x[row + i + e];
                if (a.counts) c[e] = a.counts[row + i + e];
                if (a.bias) bias[e] = a.bias[i + e];
            }
        }
        f32x4 o;
#pragma unroll
        for (uint32_t e = 0; e < 4; e++) {
            o[e] = lg_value(a, x[e], c[e], bias[e], bits >> e & 1);
            if (e < n) lg_better(b, o[e], i + e);
        }
        if (V4) *(f32x4 *)(a.out + row + i) = o;
        else
#pragma unroll
            for (uint32_t e = 0; e < 4; e++)
                if (e < n) a.out[row + i + e] = o[e];
    }
    b = lg_fold(b);
    if (threadIdx.x == 0) {
        if (gridDim.x == 1) a.token[r] = b.i;
        else part[r * gridDim.x + blockIdx.x] = b;
    }
}
__global__ void __launch_bounds__(TPB) k_logits_token(const lg_best *part, uint32_t parts, uint32_t *token) {
    lg_best b = {-INFINITY, LG_NONE};
    if (threadIdx.x < parts) b = part[(uint64_t)blockIdx.x * parts + threadIdx.x];
    b = lg_fold(b);
    if (threadIdx.x == 0) token[blockIdx.x] = b.i;
}

// parts of a row: one per 4 TPB ids, until the rows together fill the chip a few times
static uint32_t lg_parts(uint32_t vocab, uint32_t rows) {
    const uint32_t need = (uint32_t)(((uint64_t)vocab + 4 * TPB - 1) / (4 * TPB)), most = max(1u, LG_WGS / rows);
    return min(min(need, most), (uint32_t)TPB);
}
extern "C" uint64_t sgk_logits_part_bytes(uint32_t vocab, uint32_t rows) { return (uint64_t)rows * lg_parts(vocab, rows) * sizeof(lg_best); }
extern "C" hipError_t sgk_logits(const sgk_logits_args *a, void *part, hipStream_t s, hipEvent_t done) {
    if (!a->vocab || !a->rows) return hipSuccess;
    const uint32_t parts = lg_parts(a->vocab, a->rows);
    const bool v4 = !(((uintptr_t)a->x | (uintptr_t)a->out | (uintptr_t)a->counts | (uintptr_t)a->bias) & 15) && a->vocab % 4 == 0;
    const dim3 grid(parts, a->rows);
    const hipEvent_t ev = parts > 1 ? NULL : done;
    if (v4) launch(k_logits<true>, grid, TPB, s, ev, *a, (lg_best *)part);
    else launch(k_logits<false>, grid, TPB, s, ev, *a, (lg_best *)part);
    if (parts > 1) launch(k_logits_token, dim3(a->rows), TPB, s, done, (const lg_best *)part, parts, a->token);
    return hipGetLastError();
}
