// pages.hip - several sequences over a paged f16 K/V cache: rows into pages,
// attention of one token a sequence over its pages with the sum of the weights
// that each row was given, and the eviction of the rows given least. Launchers
// are declared in kernels.h; their host checks are in hip.c.
//
// Slot j of sequence s lies in page table[s][j / page] at row j % page; a page
// holds [page][n_kv][hd]. A page number outside the pool is never followed:
// its slots are not there. Every other size that comes from device memory
// (lengths, first slots, counts) is brought into its range before use.
#include "devutil.h"
#include "kernels.h"

typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));

// The row of the pool that slot j of sequence s lies in, or -1.
__device__ __forceinline__ int64_t page_row(const sgk_pages &c, uint32_t s, uint32_t j) {
    const uint32_t p = (uint32_t)c.table[(uint64_t)s * c.width + (j >> c.log)];
    return p < c.pages ? (int64_t)(((uint64_t)p << c.log) + (j & ((1u << c.log) - 1))) : -1;
}
__device__ __forceinline__ uint32_t page_len(const sgk_pages &c, const int32_t *lens, uint32_t s) {
    return min((uint32_t)max(lens[s], 0), c.width << c.log);
}

// ---------------------------------------------------------------------------
// Store: 8 dims of K and of V per thread, rounded to f16 (nearest even).
// ---------------------------------------------------------------------------
__device__ __forceinline__ f16x8 half8(const float *p, bool al) {
    const f32x4 a = ld4(p, al), b = ld4(p + 4, al);
    f16x8 r;
#pragma unroll
    for (int e = 0; e < 4; e++) { r[e] = (_Float16)a[e]; r[4 + e] = (_Float16)b[e]; }
    return r;
}
// A row's units (8 dims) go to 2^wl lanes, TPB >> wl rows a workgroup.
__global__ void __launch_bounds__(TPB) k_page_store(sgk_page_store_args a, uint32_t wl, int al) {
    const uint32_t t = threadIdx.x, units = a.c.n_kv * (a.c.hd / 8), s = blockIdx.y;
    const uint64_t cap = (uint64_t)a.c.width << a.c.log;
    for (uint64_t i = (uint64_t)blockIdx.x * (TPB >> wl) + (t >> wl); i < a.n; i += (uint64_t)gridDim.x * (TPB >> wl)) {
        const int64_t first = a.span[3 * s], rows = a.span[3 * s + 1], slot = first + (int64_t)i;
        if ((int64_t)i >= rows || first < 0 || slot >= (int64_t)cap) continue;
        const int64_t to = page_row(a.c, s, (uint32_t)slot);
        if (to < 0) continue;
        const uint64_t from = ((uint64_t)s * a.n + i) * a.stride;
        for (uint32_t u = t & ((1u << wl) - 1); u < units; u += 1u << wl) {
            const f16x8 kv = half8(a.k + from + 8 * u, al), vv = half8(a.v + from + 8 * u, al);
            *(f16x8 *)(a.c.k + ((uint64_t)to * units + u) * 8) = kv;
            *(f16x8 *)(a.c.v + ((uint64_t)to * units + u) * 8) = vv;
            if (u % (a.c.hd / 8) == 0) {
                const uint64_t at = ((uint64_t)s * a.c.n_kv + u / (a.c.hd / 8)) * cap + (uint64_t)slot;
                if (a.weight) a.weight[at] = 0.0f;
                if (a.pos) a.pos[at] = (int32_t)((uint32_t)a.span[3 * s + 2] + (uint32_t)i);
            }
        }
    }
}
extern "C" hipError_t sgk_page_store(const sgk_page_store_args *a, hipStream_t s, hipEvent_t done) {
    const uint32_t units = a->c.n_kv * (a->c.hd / 8);
    uint32_t wl = 0;
    while (wl < 8 && (1u << wl) < units) wl++;
    const uint64_t need = ((uint64_t)a->n + (TPB >> wl) - 1) / (TPB >> wl);
    const int al = !(((uintptr_t)a->k | (uintptr_t)a->v) & 15) && a->stride % 4 == 0;
    launch(k_page_store, dim3((uint32_t)(need < 1u << 20 ? need : 1u << 20), a->c.n_seq), TPB, s, done, *a, wl, al);
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Attention. A workgroup takes AP_SLOTS slots of one sequence and kv head: the
// scores of a slot by a thread, the weighted values of a dim by a thread. Each
// part leaves its maximum, its sum and its weighted values, and the scores where
// the weights are wanted; the join brings the parts together.
// ---------------------------------------------------------------------------
#define AP_SLOTS 256u
struct ap_part { float *m, *l, *acc, *score; uint32_t parts; };     // [seq][head][part], acc x hd; score [seq][head][cap]

__global__ void __launch_bounds__(TPB) k_attn_paged(sgk_attn_paged_args a, ap_part w) {
    __shared__ float qs[16][256], ps[16][AP_SLOTS], red[16][2];
    const uint32_t t = threadIdx.x, part = blockIdx.x, h = blockIdx.y, s = blockIdx.z, hd = a.c.hd, g = a.n_heads / a.c.n_kv;
    const uint32_t len = page_len(a.c, a.lens, s), j = part * AP_SLOTS + t;
    const uint64_t cap = (uint64_t)a.c.width << a.c.log, wide = (uint64_t)a.c.n_kv * hd;
    if (part * AP_SLOTS >= len) return;
    for (uint32_t i = t; i < g * hd; i += TPB) qs[i / hd][i % hd] = a.q[((uint64_t)s * a.n_heads + h * g + i / hd) * a.q_stride + i % hd];
    __shared__ int64_t rowat[AP_SLOTS];
    const int64_t row = j < len ? page_row(a.c, s, j) : -1;
    rowat[t] = row;
    __syncthreads();
    float sc[16];
    for (uint32_t c = 0; c < 16; c++) sc[c] = 0.0f;
    if (row >= 0) {
        const _Float16 *k = (const _Float16 *)a.c.k + (uint64_t)row * wide + h * hd;
        for (uint32_t d = 0; d < hd; d++) {
            const float x = (float)k[d];
            for (uint32_t c = 0; c < 16; c++) if (c < g) sc[c] = fmaf(x, qs[c][d], sc[c]);
        }
    }
    for (uint32_t c = 0; c < 16; c++)
        if (c < g) {
            const float x = row >= 0 ? sc[c] * a.scale : -INFINITY;
            ps[c][t] = x;
            if (w.score && j < len) w.score[((uint64_t)s * a.n_heads + h * g + c) * cap + j] = x;
        }
    __syncthreads();
    if (t < g) {
        float m = -INFINITY, l = 0.0f;
        for (uint32_t i = 0; i < AP_SLOTS; i++) m = ps[t][i] > m || ps[t][i] != ps[t][i] ? ps[t][i] : m;
        for (uint32_t i = 0; i < AP_SLOTS; i++) {
            const float p = rowat[i] >= 0 ? expf(ps[t][i] - m) : 0.0f;
            ps[t][i] = p;
            l += p;
        }
        const uint64_t at = ((uint64_t)s * a.n_heads + h * g + t) * w.parts + part;
        w.m[at] = m;
        w.l[at] = l;
    }
    __syncthreads();
    if (t < hd) {
        float o[16];
        for (uint32_t c = 0; c < 16; c++) o[c] = 0.0f;
        for (uint32_t i = 0; i < AP_SLOTS; i++) {
            if (rowat[i] < 0) continue;
            const float v = (float)((const _Float16 *)a.c.v)[(uint64_t)rowat[i] * wide + h * hd + t];
            for (uint32_t c = 0; c < 16; c++) if (c < g) o[c] = fmaf(ps[c][i], v, o[c]);
        }
        for (uint32_t c = 0; c < 16; c++)
            if (c < g) w.acc[(((uint64_t)s * a.n_heads + h * g + c) * w.parts + part) * hd + t] = o[c];
    }
}
// A workgroup per sequence and query head: the parts' sum.
__global__ void __launch_bounds__(TPB) k_attn_paged_join(sgk_attn_paged_args a, ap_part w) {
    const uint32_t t = threadIdx.x, c = blockIdx.x, s = blockIdx.y, hd = a.c.hd;
    const uint32_t len = page_len(a.c, a.lens, s), n = (len + AP_SLOTS - 1) / AP_SLOTS;
    const uint64_t at = ((uint64_t)s * a.n_heads + c) * w.parts;
    float m = -INFINITY, l = 0.0f, o = 0.0f;
    for (uint32_t i = 0; i < n; i++) m = w.m[at + i] > m || w.m[at + i] != w.m[at + i] ? w.m[at + i] : m;
    for (uint32_t i = 0; i < n; i++) {
        const float f = w.m[at + i] == -INFINITY ? 0.0f : expf(w.m[at + i] - m);
        l = fmaf(f, w.l[at + i], l);
        if (t < hd && f != 0.0f) o = fmaf(f, w.acc[(at + i) * hd + t], o);
    }
    if (t < hd) a.out[((uint64_t)s * a.n_heads + c) * hd + t] = m == -INFINITY ? 0.0f : o / l;
    if (w.score && t == 0) { w.m[at] = m; w.l[at] = l; }
}
__global__ void __launch_bounds__(TPB) k_attn_paged_weights(sgk_attn_paged_args a, ap_part w) {
    const uint32_t h = blockIdx.y, s = blockIdx.z, g = a.n_heads / a.c.n_kv, len = page_len(a.c, a.lens, s);
    const uint64_t cap = (uint64_t)a.c.width << a.c.log;
    for (uint32_t j = blockIdx.x * TPB + threadIdx.x; j < len; j += gridDim.x * TPB) {
        const uint64_t at = ((uint64_t)s * a.c.n_kv + h) * cap + j;
        float sum = 0.0f;
        if (page_row(a.c, s, j) >= 0)
            for (uint32_t c = h * g; c < h * g + g; c++) {
                const uint64_t r = (uint64_t)s * a.n_heads + c;
                sum += expf(w.score[r * cap + j] - w.m[r * w.parts]) / w.l[r * w.parts];
            }
        a.weight_out[at] = (a.weight ? a.weight[at] : 0.0f) + sum;
    }
}
static ap_part ap_plan(const sgk_attn_paged_args *a, void *scratch, uint64_t *bytes) {
    const uint64_t rows = (uint64_t)a->c.n_seq * a->n_heads, cap = (uint64_t)a->c.width << a->c.log;
    const uint64_t parts = (cap + AP_SLOTS - 1) / AP_SLOTS;
    float *f = (float *)scratch;
    *bytes = 4 * (rows * parts * (2 + a->c.hd) + (a->weight_out ? rows * cap : 0));
    return (ap_part){f, f + rows * parts, f + 2 * rows * parts, a->weight_out ? f + rows * parts * (2 + a->c.hd) : NULL, (uint32_t)parts};
}
extern "C" uint64_t sgk_attn_paged_scratch(const sgk_attn_paged_args *a) {
    uint64_t bytes;
    ap_plan(a, NULL, &bytes);
    return bytes;
}
extern "C" hipError_t sgk_attn_paged(const sgk_attn_paged_args *a, void *scratch, hipStream_t s, hipEvent_t done) {
    uint64_t bytes;
    const ap_part w = ap_plan(a, scratch, &bytes);
    launch(k_attn_paged, dim3(w.parts, a->c.n_kv, a->c.n_seq), TPB, s, (hipEvent_t)NULL, *a, w);
    launch(k_attn_paged_join, dim3(a->n_heads, a->c.n_seq), TPB, s, a->weight_out ? (hipEvent_t)NULL : done, *a, w);
    if (a->weight_out) launch(k_attn_paged_weights, dim3(w.parts < 256 ? w.parts : 256, a->c.n_kv, a->c.n_seq), TPB, s, done, *a, w);
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Eviction. The order of a (sequence, kv head)'s slots: recent ones first, then
// by weight, then the lower slot; the first `keep` stay. A workgroup finds the
// keep-th key by its digits (8 bits a pass over the slots), then lists the freed
// slots below keep and the kept ones from keep on, both rising, and a second
// launch moves the n-th of these to the n-th of those. No row that is read is
// written, so the moves need no order.
// ---------------------------------------------------------------------------
#define EV_THREADS 1024
struct ev_list { uint32_t *hole, *mover, *n; };      // [row][keep] twice, [row]

// Rising with the order: 0xFFFFFFFF recent, 0 NaN.
__device__ __forceinline__ uint32_t ev_key(float w, int32_t pos, int64_t after) {
    const uint32_t b = __float_as_uint(w + 0.0f);       // -0 as 0
    const uint32_t key = b & 0x80000000u ? ~b : b | 0x80000000u;
    return (int64_t)pos > after ? 0xFFFFFFFFu : w != w ? 0u : key;
}
// exclusive prefix sum over the workgroup, and the total
__device__ __forceinline__ uint32_t ev_scan(uint32_t v, uint32_t *total, uint32_t *tmp) {
    const uint32_t t = threadIdx.x;
    uint32_t x = v;
    for (uint32_t d = 1; d < 64; d <<= 1) {
        const uint32_t y = __shfl_up(x, d);
        if ((t & 63) >= d) x += y;
    }
    __syncthreads();
    if ((t & 63) == 63) tmp[t >> 6] = x;
    __syncthreads();
    uint32_t before = 0, all = 0;
    for (uint32_t i = 0; i < EV_THREADS / 64; i++) {
        if (i < t >> 6) before += tmp[i];
        all += tmp[i];
    }
    *total = all;
    return before + x - v;
}
__global__ void __launch_bounds__(EV_THREADS) k_page_evict_select(sgk_page_evict_args a, ev_list w) {
    __shared__ uint32_t hist[256], tmp[EV_THREADS / 64], pick[2];
    __shared__ int32_t lastp[EV_THREADS / 64];
    const uint32_t t = threadIdx.x, h = blockIdx.x, s = blockIdx.y, len = page_len(a.c, a.lens, s);
    const uint64_t cap = (uint64_t)a.c.width << a.c.log, row = (uint64_t)s * a.c.n_kv + h;
    const float *wt = a.weight + row * cap;
    const int32_t *ps = a.pos + row * cap;
    const uint32_t keep = min(a.keep, len);
    if (a.weight_out != a.weight) for (uint32_t j = t; j < keep; j += EV_THREADS) a.weight_out[row * cap + j] = wt[j];
    if (a.pos_out != a.pos) for (uint32_t j = t; j < keep; j += EV_THREADS) a.pos_out[row * cap + j] = ps[j];
    if (t == 0) w.n[row] = 0;
    if (len <= a.keep) return;
    int32_t last = INT32_MIN;
    for (uint32_t j = t; j < len; j += EV_THREADS) last = max(last, ps[j]);
    for (uint32_t d = 1; d < 64; d <<= 1) last = max(last, __shfl_xor(last, d));
    if ((t & 63) == 0) lastp[t >> 6] = last;
    __syncthreads();
    for (uint32_t i = 0; i < EV_THREADS / 64; i++) last = max(last, lastp[i]);
    const int64_t after = (int64_t)last - a.recent;
    uint32_t prefix = 0, left = keep;           // of slots with the prefix, `left` stay
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (t < 256) hist[t] = 0;
        __syncthreads();
        for (uint32_t j = t; j < len; j += EV_THREADS) {
            const uint32_t key = ev_key(wt[j], ps[j], after);
            if (shift == 24 || key >> (shift + 8) == prefix >> (shift + 8)) atomicAdd(&hist[key >> shift & 255], 1u);
        }
        __syncthreads();
        if (t == 0) {
            uint32_t b = 255;
            while (hist[b] < left) left -= hist[b--];
            pick[0] = prefix | b << shift;
            pick[1] = left;
        }
        __syncthreads();
        prefix = pick[0];
        left = pick[1];
    }
    // prefix is the keep-th key; `left` of its slots stay, the lowest
    uint32_t ties = 0, holes = 0, movers = 0;
    for (uint32_t j0 = 0; j0 < len; j0 += EV_THREADS) {
        const uint32_t j = j0 + t, key = j < len ? ev_key(wt[j], ps[j], after) : 0;
        uint32_t n;
        const uint32_t tie = j < len && key == prefix, rank = ties + ev_scan(tie, &n, tmp);
        ties += n;
        const bool kept = j < len && (key > prefix || (tie && rank < left));
        const uint32_t hole = j < keep && !kept, hr = holes + ev_scan(hole, &n, tmp);
        holes += n;
        const uint32_t mover = j >= keep && kept, mr = movers + ev_scan(mover, &n, tmp);
        movers += n;
        if (hole) w.hole[row * a.keep + hr] = j;
        if (mover) w.mover[row * a.keep + mr] = j;
    }
    if (t == 0) w.n[row] = holes;
}
__global__ void __launch_bounds__(TPB) k_page_evict_move(sgk_page_evict_args a, ev_list w) {
    const uint32_t h = blockIdx.y, s = blockIdx.z, units = a.c.hd / 8;
    const uint64_t cap = (uint64_t)a.c.width << a.c.log, row = (uint64_t)s * a.c.n_kv + h, wide = (uint64_t)a.c.n_kv * units;
    const uint64_t n = (uint64_t)w.n[row] * units;
    for (uint64_t i = (uint64_t)blockIdx.x * TPB + threadIdx.x; i < n; i += (uint64_t)gridDim.x * TPB) {
        const uint32_t u = (uint32_t)(i % units), to = w.hole[row * a.keep + i / units], from = w.mover[row * a.keep + i / units];
        if (u == 0) {
            a.weight_out[row * cap + to] = a.weight[row * cap + from];
            a.pos_out[row * cap + to] = a.pos[row * cap + from];
        }
        const int64_t x = page_row(a.c, s, from), y = page_row(a.c, s, to);
        if (x < 0 || y < 0) continue;
        const uint64_t xi = (uint64_t)x * wide + h * units + u, yi = (uint64_t)y * wide + h * units + u;
        ((u16x8 *)a.c.k)[yi] = ((const u16x8 *)a.c.k)[xi];
        ((u16x8 *)a.c.v)[yi] = ((const u16x8 *)a.c.v)[xi];
    }
}
extern "C" uint64_t sgk_page_evict_scratch(const sgk_page_evict_args *a) {
    return 4 * (uint64_t)a->c.n_seq * a->c.n_kv * (2 * (uint64_t)a->keep + 1);
}
extern "C" hipError_t sgk_page_evict(const sgk_page_evict_args *a, void *scratch, hipStream_t s, hipEvent_t done) {
    const uint64_t rows = (uint64_t)a->c.n_seq * a->c.n_kv, each = rows * a->keep;
    uint32_t *u = (uint32_t *)scratch;
    const ev_list w = {u, u + each, u + 2 * each};
    launch(k_page_evict_select, dim3(a->c.n_kv, a->c.n_seq), EV_THREADS, s, (hipEvent_t)NULL, *a, w);
    const uint64_t b = ((uint64_t)a->keep * (a->c.hd / 8) + TPB - 1) / TPB;
    launch(k_page_evict_move, dim3((uint32_t)(b < 256 ? b : 256), a->c.n_kv, a->c.n_seq), TPB, s, done, *a, w);
    return hipGetLastError();
}
