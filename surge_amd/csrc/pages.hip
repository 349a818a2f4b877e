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

// An address that a wave's lanes share, as the scalar base of its loads.
__device__ __forceinline__ const char *uniform(const char *p) {
    const uint64_t a = (uint64_t)(uintptr_t)p;
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)a), hi = __builtin_amdgcn_readfirstlane((uint32_t)(a >> 32));
    return (const char *)(const __attribute__((address_space(1))) char *)(uintptr_t)((uint64_t)hi << 32 | lo);
}
// The row of the pool that slot j of sequence s lies in, or -1.
__device__ __forceinline__ int64_t page_row(const sgk_pages &c, uint32_t s, uint32_t j) {
    const uint32_t p = (uint32_t)c.table[(uint64_t)s * c.width + (j >> c.log)];
    return p < c.pages ? (int64_t)(((uint64_t)p << c.log) + (j & ((1u << c.log) - 1))) : -1;
}
__device__ __forceinline__ uint32_t page_len(const sgk_pages &c, const int32_t *lens, uint32_t s) {
    return min((uint32_t)max(((const scalar_i32 *)(uintptr_t)lens)[s], 0), c.width << c.log);
}

// ---------------------------------------------------------------------------
// Store: 8 dims of K and of V per thread, rounded to f16 (nearest even). Bound by
// memory (8190 rows of 4 x 256, 100 MB read and written: 20.4 us, 4.9 TB/s, as a
// copy) or, a few rows, by one trip to the spans, the table and the rows (3.1 us).
// Asking for the data before the span and the page are known changes neither
// (3.0; 21.2).
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
// Attention. Parts of the sequences, a workgroup each per kv head; in a part the
// waves take steps of 32 slots in turn, K and V straight from the pages into the
// matrix instructions' operands, with a running maximum and sum per wave. Their
// results are added in LDS, those of a sequence's parts by a second launch.
//
// Scores^T = K q^T, 16 slots x 16 heads a product: lane (r, g) = (l % 16, l / 16)
// loads slot r, dims 32 j + 8 g ..+7, and gets the scores of head r at slots
// 4 g ..+3. Two such tiles make the 32 slots of out^T = V^T p^T, whose k index
// 8 g + e stands for slot 4 g + e of the first tile (e < 4) or the second: a lane
// has its own scores as operand. Of V it loads those eight rows, 8 dims each
// (dims 8 r ..+7 of 128; 4 at head_dim 64), and dim 8 r + j of them is row r of
// the j-th product, one byte permutation per two values.
//
// q is split into three f16, scaled so that its head's largest element is 2^14 to
// 2^15: what is left of an element is below 2^-25 then (half of f16's smallest), 2^-39
// of the largest, and nothing of elements from 2^-15 of it on. p is split into two
// (2^-22). So products are exact or nearly so, and sums are f32.
//
// Parts: T steps in all and `most` parts a kv head wanted give parts of `per` =
// ceil(T / most) steps, a multiple of the waves, the same on every workgroup; a
// sequence of n steps has ceil(n / per) of them, so there are at most most + n_seq,
// and its steps are spread over them evenly (64 sequences of 1800 to 2300 slots: 78
// us, 94 with a short last part).
//
// Bound by reading K and V once: a step's products are a tenth of its time on the
// matrix units. A wave has its next step's K and V under way all the time, 8 to 32 KB,
// and 32 slots a step are what its registers hold at head_dim 256 (242 of 256). What
// is read once goes past the caches' order of use (non-temporal: 262000 slots of 4 x
// 256 178 us against 185, then with two workgroups a CU). 175 us for those 1073 MB, 6.1
// TB/s (a plain read of as much 181), 78 for 64 sequences' 401 MB, 51 for 16 of 91 to
// 16411 slots, 231 MB. Past 64 sequences the plan is a launch of its own (3.9 us). About 9
// us of each are the chain that a short call consists of (4 sequences of 57 to 700
// slots, 9.2): lengths, table, rows, two products, the waves' sums.
// ---------------------------------------------------------------------------
#define AP_STEP 32u
#define AP_WAVES 4u
#define AP_MOST 1024u      // parts of a sequence, at most
#define AP_P2 14            // p is held times 2^14, so that f16's subnormals start at 2^-28

struct ap_part {
    float *m, *l, *acc;     // [part][head], acc x hd
    float *score;           // [seq][head][cap], or NULL
    uint32_t *plan;         // [n_seq + 1] first parts, then [parts] sequences; NULL up to 64 sequences
    uint32_t most, parts;
};

__device__ __forceinline__ uint32_t ap_steps(const sgk_attn_paged_args &a, uint32_t s) { return (page_len(a.c, a.lens, s) + AP_STEP - 1) / AP_STEP; }
__device__ __forceinline__ uint32_t ap_per(uint64_t total, uint32_t most) { return (max((uint32_t)((total + most - 1) / most), 1u) + AP_WAVES - 1) / AP_WAVES * AP_WAVES; }
struct ap_where { uint32_t s, first, n, per; };      // sequence (n_seq: none), its first part and their number
// Of part x (by_part) or of sequence x.
__device__ __forceinline__ ap_where ap_find(const sgk_attn_paged_args &a, const ap_part &w, uint32_t x, bool by_part) {
    const uint32_t ns = a.c.n_seq;
    if (w.plan) {
        const uint32_t all = w.plan[ns], s = !by_part ? x : x < all ? w.plan[ns + 2 + x] : ns;
        if (s >= ns) return (ap_where){ns, 0, 0, 0};
        return (ap_where){s, w.plan[s], w.plan[s + 1] - w.plan[s], w.plan[ns + 1]};
    }
    if (ns == 1) {
        const uint32_t st = ap_steps(a, 0), per = ap_per(st, w.most), n = (st + per - 1) / per;
        return (ap_where){by_part && x >= n ? 1u : 0u, 0, n, per};
    }
    const uint32_t l = threadIdx.x & 63, st = l < ns ? ap_steps(a, l) : 0;
    const uint32_t per = ap_per((uint32_t)__builtin_amdgcn_readlane((int)wave_scan(st), 63), w.most);     // 64 x 2^25 steps at most
    const uint32_t n = (st + per - 1) / per, to = wave_scan(n);
    const uint32_t s = by_part ? (uint32_t)__popcll(__builtin_amdgcn_ballot_w64(to <= x)) : x;
    if (s >= ns) return (ap_where){ns, 0, 0, 0};
    const uint32_t e = (uint32_t)__builtin_amdgcn_readlane((int)to, (int)s), c = (uint32_t)__builtin_amdgcn_readlane((int)n, (int)s);
    return (ap_where){s, e - c, c, per};
}
// The plan of more than 64 sequences: [n_seq] all parts, [n_seq + 1] steps a part.
__global__ void __launch_bounds__(1024) k_attn_paged_plan(sgk_attn_paged_args a, ap_part w) {
    __shared__ uint64_t tot[16];
    __shared__ uint32_t sub[16];
    const uint32_t t = threadIdx.x, ns = a.c.n_seq;
    uint64_t sum = 0;
    for (uint32_t s = t; s < ns; s += 1024) sum += ap_steps(a, s);
    for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
    if ((t & 63) == 0) tot[t >> 6] = sum;
    __syncthreads();
    sum = 0;
    for (int i = 0; i < 16; i++) sum += tot[i];
    const uint32_t per = ap_per(sum, w.most);
    uint32_t at = 0;
    for (uint32_t s0 = 0; s0 < ns; s0 += 1024) {
        const uint32_t s = s0 + t, n = s < ns ? (ap_steps(a, s) + per - 1) / per : 0, to = wave_scan(n);
        __syncthreads();
        if ((t & 63) == 63) sub[t >> 6] = to;
        __syncthreads();
        uint32_t first = at + to - n;
        for (uint32_t i = 0; i < 16; i++) {
            if (i < t >> 6) first += sub[i];
            at += sub[i];
        }
        if (s < ns) {
            w.plan[s] = first;
            for (uint32_t i = 0; i < n; i++) w.plan[ns + 2 + first + i] = s;
        }
    }
    if (t == 0) { w.plan[ns] = at; w.plan[ns + 1] = per; }
}

__device__ __forceinline__ f16x2 pair_of(uint32_t b, uint32_t a, bool high) {      // the low or the high halves of two dwords
    union { uint32_t u; f16x2 h; } r;
    r.u = __builtin_amdgcn_perm(b, a, high ? 0x07060302u : 0x05040100u);
    return r.h;
}

template <int HD>
__global__ void __launch_bounds__(AP_WAVES * 64, 2) k_attn_paged(sgk_attn_paged_args a, ap_part w, int al) {
    constexpr int NJ = HD / 32, NT = HD / 16, VD = HD == 64 ? 4 : 8, NC = HD / (16 * VD);      // VD dims a lane and chunk of V
    typedef uint32_t vrow __attribute__((ext_vector_type(VD / 2)));
    extern __shared__ __align__(16) char lds[];
    f16x8 (*qs)[NJ][64] = (f16x8 (*)[NJ][64])lds;
    const uint32_t t = threadIdx.x, l = t & 63, r = l & 15, g = l >> 4, wv = __builtin_amdgcn_readfirstlane(t >> 6);
    const uint32_t h = blockIdx.x, part = blockIdx.y, grp = a.n_heads / a.c.n_kv;
    const ap_where me = ap_find(a, w, part, true);
    if (me.s >= a.c.n_seq) return;
    const uint32_t s = me.s, len = page_len(a.c, a.lens, s), all = (len + AP_STEP - 1) / AP_STEP;
    // the sequence's steps, evenly over its parts (a multiple of the waves)
    const uint32_t each = ((all + me.n - 1) / me.n + AP_WAVES - 1) / AP_WAVES * AP_WAVES;
    const uint32_t st0 = min((part - me.first) * each, all), st1 = min(st0 + each, all);
    const uint64_t wide = (uint64_t)a.c.n_kv * HD, cap = (uint64_t)a.c.width << a.c.log;
    const scalar_i32 *table = (const scalar_i32 *)(uintptr_t)(a.c.table + (uint64_t)s * a.c.width);

    // q of head r, dims 32 j + 8 g ..+7: all of it for its largest element, the j that are the wave's mod the waves as three f16
    float qx[NJ][8];
    {
        const float *q = a.q + ((uint64_t)s * a.n_heads + h * grp + min(r, grp - 1)) * a.q_stride + 8 * g;
        if (al) {
#pragma unroll
            for (int j = 0; j < NJ; j++)
#pragma unroll
                for (int z = 0; z < 2; z++) {
                    const f32x4 y = *(const f32x4 *)(q + 32 * j + 4 * z);
#pragma unroll
                    for (int e = 0; e < 4; e++) qx[j][4 * z + e] = y[e];
                }
        } else {
#pragma unroll
            for (int j = 0; j < NJ; j++)
#pragma unroll
                for (int e = 0; e < 8; e++) qx[j][e] = q[32 * j + e];
        }
    }
    // a half step's rows: whether they are there, and where in the pools (uniform); slots behind the last: its page
    struct half_at { bool ok; uint64_t off; };
    auto at = [&](uint32_t j) -> half_at {
        const uint32_t p = (uint32_t)table[min(j, len - 1) >> a.c.log];
        const bool ok = p < a.c.pages;
        return (half_at){ok && j < len, ((((uint64_t)(ok ? p : 0) << a.c.log) + (j & ((1u << a.c.log) - 1))) * wide + h * HD) * 2};
    };
    f16x8 kf[2][NJ];
    const uint32_t koff = (r * (uint32_t)wide + 8 * g) * 2;
    uint32_t voff[4];
#pragma unroll
    for (int e = 0; e < 4; e++) voff[e] = ((4 * g + e) * (uint32_t)wide + VD * r) * 2;
    auto load_k = [&](const half_at (&p)[2]) {
#pragma unroll
        for (int z = 0; z < 2; z++)
#pragma unroll
            for (int j = 0; j < NJ; j++) kf[z][j] = __builtin_nontemporal_load((const f16x8 *)(uniform((const char *)a.c.k + p[z].off) + koff + 64 * j));
    };
    vrow vf[NC][8];
    auto load_v = [&](const half_at (&p)[2]) {
#pragma unroll
        for (int e = 0; e < 8; e++)
#pragma unroll
            for (int c = 0; c < NC; c++)
                vf[c][e] = __builtin_nontemporal_load((const vrow *)(uniform((const char *)a.c.v + p[e / 4].off) + voff[e % 4] + 32 * VD * c));
    };
    half_at now[2] = {at((st0 + wv) * AP_STEP), at((st0 + wv) * AP_STEP + 16)};
    if (st0 + wv < st1) { load_k(now); load_v(now); }
    __builtin_amdgcn_sched_barrier(0);
    float f1;
    {
        float am = 0.0f;
#pragma unroll
        for (int j = 0; j < NJ; j++)
#pragma unroll
            for (int e = 0; e < 8; e++) am = fmaxf(am, fabsf(qx[j][e]));
        am = fmaxf(am, swap16f(am));
        am = fmaxf(am, swap32f(am));
        const int ex = am > 0.0f && am < INFINITY ? __builtin_amdgcn_frexp_expf(am) : 0;
        f1 = __builtin_amdgcn_ldexpf(a.scale, ex - 15);
#pragma unroll
        for (int j = 0; j < NJ; j++) {
            if (j % AP_WAVES != wv) continue;
            f16x8 p[3];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                float y = __builtin_amdgcn_ldexpf(qx[j][e], 15 - ex);
#pragma unroll
                for (int z = 0; z < 3; z++) {
                    p[z][e] = (_Float16)y;
                    y -= (float)p[z][e];
                }
            }
#pragma unroll
            for (int z = 0; z < 3; z++) qs[z][j][l] = p[z];
        }
    }
    __syncthreads();

    float m = -INFINITY, sum = 0.0f;
    f32x4 o[NT];
#pragma unroll
    for (int i = 0; i < NT; i++) o[i] = (f32x4){0, 0, 0, 0};
    for (uint32_t st = st0 + wv; st < st1; st += AP_WAVES) {
        const uint32_t j0 = st * AP_STEP;
        const half_at next[2] = {at(j0 + AP_WAVES * AP_STEP), at(j0 + AP_WAVES * AP_STEP + 16)};
        asm volatile("" ::: "memory");      // q's parts are read again every step, not kept in registers
        float x[8];
        f32x4 d[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
        for (int y = 2; y >= 0; y--)
#pragma unroll
            for (int j = 0; j < NJ; j++) {
                const f16x8 qf = qs[y][j][l];
#pragma unroll
                for (int z = 0; z < 2; z++) d[z] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[z][j], qf, d[z], 0, 0, 0);
            }
#pragma unroll
        for (int z = 0; z < 2; z++)
#pragma unroll
            for (int e = 0; e < 4; e++) x[4 * z + e] = now[z].ok && j0 + 16 * z + 4 * g + e < len ? d[z][e] * f1 : -INFINITY;
        __builtin_amdgcn_sched_barrier(0);
        if (st + AP_WAVES < st1) load_k(next);
        __builtin_amdgcn_sched_barrier(0);
        if (w.score && r < grp) {
            float *sc = w.score + ((uint64_t)s * a.n_heads + h * grp + r) * cap + j0 + 4 * g;
#pragma unroll
            for (int z = 0; z < 2; z++)
                if (j0 + 16 * z < cap) *(f32x4 *)(sc + 16 * z) = (f32x4){x[4 * z], x[4 * z + 1], x[4 * z + 2], x[4 * z + 3]};
        }
        float tm = x[0];
#pragma unroll
        for (int e = 1; e < 8; e++) tm = fmaxf(tm, x[e]);
        tm = fmaxf(tm, swap16f(tm));
        tm = fmaxf(tm, swap32f(tm));
        if (__builtin_amdgcn_ballot_w64(tm > m)) {
            const float mn = fmaxf(m, tm), f = m > -INFINITY ? exp2f((m - mn) * 1.44269504f) : 0.0f;
            sum *= f;
#pragma unroll
            for (int i = 0; i < NT; i++) o[i] *= f;
            m = mn;
        }
        const float mm = m > -INFINITY ? m : 0.0f;
        f16x8 ph, pl;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float p = exp2f((x[e] - mm) * 1.44269504f) * (float)(1 << AP_P2);
            sum += p;
            ph[e] = (_Float16)p;
            pl[e] = (_Float16)(p - (float)ph[e]);
        }
        if (!now[0].ok || !now[1].ok || j0 + AP_STEP > len) {       // rows that are not there may hold anything
#pragma unroll
            for (int e = 0; e < 8; e++)
#pragma unroll
                for (int c = 0; c < NC; c++)
                    if (!now[e / 4].ok || j0 + 16 * (e / 4) + 4 * g + e % 4 >= len) vf[c][e] = (vrow)0;
        }
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int j = 0; j < VD; j++) {
                union { f16x2 p[4]; f16x8 v; } u;
#pragma unroll
                for (int e = 0; e < 4; e++) u.p[e] = pair_of(vf[c][2 * e + 1][j / 2], vf[c][2 * e][j / 2], j & 1);
                f32x4 &d = o[c * VD + j];
                d = __builtin_amdgcn_mfma_f32_16x16x32_f16(u.v, pl, d, 0, 0, 0);
                d = __builtin_amdgcn_mfma_f32_16x16x32_f16(u.v, ph, d, 0, 0, 0);
            }
        __builtin_amdgcn_sched_barrier(0);
        if (st + AP_WAVES < st1) load_v(next);
        now[0] = next[0];
        now[1] = next[1];
    }
    sum += swap16f(sum);
    sum += swap32f(sum);

    // the waves' results, added: o[c VD + j][i] of lane (r, g) is head r, dim 16 VD c + VD (4 g + i) + j
    __syncthreads();
    float *wm = (float *)lds, *wl = wm + AP_WAVES * 16, *wo = wl + AP_WAVES * 16;       // [wave][16] twice, [wave][grp][HD + 4]
    if (g == 0) { wm[wv * 16 + r] = m; wl[wv * 16 + r] = sum; }
    if (r < grp) {
        float *d = wo + (wv * grp + r) * (HD + 4) + 4 * g * VD;
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < VD; j += 4)
                    *(f32x4 *)(d + 16 * VD * c + VD * i + j) = (f32x4){o[c * VD + j][i], o[c * VD + j + 1][i], o[c * VD + j + 2][i], o[c * VD + j + 3][i]};
    }
    __syncthreads();
    for (uint32_t i = t; i < grp * (HD / 4); i += AP_WAVES * 64) {
        const uint32_t c = i / (HD / 4), d = i % (HD / 4) * 4;
        float mx = -INFINITY, lx = 0.0f;
        f32x4 ox = {0, 0, 0, 0};
#pragma unroll
        for (uint32_t v = 0; v < AP_WAVES; v++) mx = fmaxf(mx, wm[v * 16 + c]);
#pragma unroll
        for (uint32_t v = 0; v < AP_WAVES; v++) {
            const float mv = wm[v * 16 + c], f = mv > -INFINITY ? exp2f((mv - mx) * 1.44269504f) : 0.0f;
            lx = fmaf(f, wl[v * 16 + c], lx);
            ox += f * *(const f32x4 *)(wo + (v * grp + c) * (HD + 4) + d);
        }
        const uint64_t at = (uint64_t)part * a.n_heads + h * grp + c;
        *(f32x4 *)(w.acc + at * HD + d) = ox;
        if (d == 0) { w.m[at] = mx; w.l[at] = lx; }
    }
}

// A head's parts, one a lane (of the first 64; the others are read when they are needed).
struct ap_lane { float m, l; };
__device__ __forceinline__ ap_lane ap_read(const ap_part &w, uint64_t at, uint32_t i, uint32_t n, uint32_t stride) {
    if (i >= n) return (ap_lane){-INFINITY, 0.0f};
    return (ap_lane){w.m[at + (uint64_t)i * stride], w.l[at + (uint64_t)i * stride]};
}
__device__ __forceinline__ float ap_factor(float mi, float m) { return mi > -INFINITY ? exp2f((mi - m) * 1.44269504f) : 0.0f; }
// The largest of the parts' maxima, and the sum of their sums under it: a wave, all lanes get them. f: the parts'
// factors, or NULL.
__device__ __forceinline__ f32x2 ap_maxsum(const ap_part &w, ap_lane x, uint64_t at, uint32_t n, uint32_t stride, float *f) {
    const uint32_t l = threadIdx.x & 63;
    float m = x.m;
    for (uint32_t i = l + 64; i < n; i += 64) m = fmaxf(m, ap_read(w, at, i, n, stride).m);
    m = wave_fmax(m);
    float sum = 0.0f;
    for (uint32_t i = l; i < n; i += 64) {
        if (i != l) x = ap_read(w, at, i, n, stride);
        const float fi = ap_factor(x.m, m);
        sum = fmaf(fi, x.l, sum);
        if (f) f[i] = fi;
    }
    return (f32x2){m, wave_fsum(sum)};
}
// A workgroup per 4 LANES dims of a query head and sequence adds the parts, four dims a lane, the parts by groups of LANES in turn.
// Where the weights are wanted, the workgroups behind take a sequence's slots, one kv head each. Whatever can be asked
// for is, before the first of it is waited for: the launch is three trips to memory long.
template <uint32_t LANES>
__global__ void __launch_bounds__(TPB) k_attn_paged_join(sgk_attn_paged_args a, ap_part w) {
    __shared__ float f[AP_MOST];
    __shared__ f32x4 red[TPB];
    __shared__ f32x2 ml[16];
    const uint32_t t = threadIdx.x, s = blockIdx.y, hd = a.c.hd, g = a.n_heads / a.c.n_kv, adders = a.n_heads * (hd / (4 * LANES));
    const ap_where me = ap_find(a, w, s, false);
    if (blockIdx.x < adders) {
        const uint32_t each = hd / (4 * LANES), head = blockIdx.x / each, d = (blockIdx.x % each * LANES + t % LANES) * 4, p0 = t / LANES;
        const uint64_t at = (uint64_t)me.first * a.n_heads + head;
        ap_lane x = {};
        if (t < 64) x = ap_read(w, at, t, me.n, a.n_heads);
        const float *acc = w.acc + at * hd + d;
        constexpr uint32_t A = 4, G = TPB / LANES;
        f32x4 o = {0, 0, 0, 0}, y[A];
#pragma unroll
        for (uint32_t i = 0; i < A; i++) y[i] = p0 + i * G < me.n ? *(const f32x4 *)(acc + (uint64_t)(p0 + i * G) * a.n_heads * hd) : (f32x4){0, 0, 0, 0};
        if (t < 64) {
            const f32x2 r = ap_maxsum(w, x, at, me.n, a.n_heads, f);
            if (t == 0) ml[0] = r;
        }
        __syncthreads();
#pragma unroll
        for (uint32_t i = 0; i < A; i++)
            if (p0 + i * G < me.n) o += f[p0 + i * G] * y[i];
#pragma unroll 4
        for (uint32_t i = p0 + A * G; i < me.n; i += G) o += f[i] * *(const f32x4 *)(acc + (uint64_t)i * a.n_heads * hd);
        red[t] = o;
        __syncthreads();
        if (t >= LANES) return;
#pragma unroll
        for (uint32_t i = 1; i < G; i++) o += red[t + i * LANES];
        const float l = ml[0][1];
#pragma unroll
        for (int e = 0; e < 4; e++) a.out[((uint64_t)s * a.n_heads + head) * hd + d + e] = l == 0.0f ? 0.0f : o[e] / l;
        return;
    }
    const uint32_t x = blockIdx.x - adders, h = x % a.c.n_kv, nb = (gridDim.x - adders) / a.c.n_kv, len = page_len(a.c, a.lens, s);
    const uint64_t cap = (uint64_t)a.c.width << a.c.log, at = ((uint64_t)s * a.c.n_kv + h) * cap, head0 = (uint64_t)me.first * a.n_heads + h * g;
    uint32_t j = (x / a.c.n_kv) * TPB + t;
    if (j - t >= len) return;
    ap_lane y[4];
#pragma unroll
    for (uint32_t i = 0; i < 4; i++)
        if (t / 64 + 4 * i < g) y[i] = ap_read(w, head0 + t / 64 + 4 * i, t & 63, me.n, a.n_heads);
    const float *sc = w.score + ((uint64_t)s * a.n_heads + h * g) * cap;
    float z[16], before = 0.0f;
    auto fetch = [&]() {
        if (j >= len) return;
#pragma unroll
        for (uint32_t c = 0; c < 16; c++)
            if (c < g) z[c] = sc[c * cap + j];
        before = a.weight ? a.weight[at + j] : 0.0f;
    };
    fetch();
#pragma unroll
    for (uint32_t i = 0; i < 4; i++) {
        const uint32_t c = t / 64 + 4 * i;
        if (c >= g) break;
        const f32x2 r = ap_maxsum(w, y[i], head0 + c, me.n, a.n_heads, NULL);
        if ((t & 63) == 0) ml[c] = (f32x2){r[0], (float)(1 << AP_P2) / r[1]};
    }
    __syncthreads();
    while (j < len) {
        float sum = 0.0f;
        // a slot that is not there has -inf for a score, and so no weight
#pragma unroll
        for (uint32_t c = 0; c < 16; c++)
            if (c < g && z[c] != -INFINITY) sum = fmaf(exp2f((z[c] - ml[c][0]) * 1.44269504f), ml[c][1], sum);
        a.weight_out[at + j] = before + sum;
        j += nb * TPB;
        fetch();
    }
}
static ap_part ap_plan(const sgk_attn_paged_args *a, char *at, uint64_t *bytes) {
    const uint64_t rows = (uint64_t)a->c.n_seq * a->n_heads, cap = (uint64_t)a->c.width << a->c.log;
    const uint64_t steps = (cap + AP_STEP - 1) / AP_STEP * a->c.n_seq;      // at most
    // Workgroups that are there together: two a CU, which even out sequences of unlike lengths, or one where a single sequence
    // is cut evenly anyway and 64 KB a CU are still asked for at once (head_dim 128; 64 has two). More of them are slower, us
    // a call: 262000 slots of 256 186 with one, 190 with two, 196 with four; 200000 of one head of 128 40, 44, 48.5 (three);
    // 8 sequences of 128 56.7 with two, 59.9 with three. A sequence's last part is short, so that n_seq - 1 more may come up.
    const uint64_t there = (uint64_t)(a->c.n_seq == 1 && a->c.hd >= 128 ? 1 : 2) * sgk_device_cus() / a->c.n_kv;
    uint64_t most = there >= 2 * a->c.n_seq ? there - (a->c.n_seq - 1) : there;
    if (most > AP_MOST) most = AP_MOST;
    if (most > (steps + AP_WAVES - 1) / AP_WAVES) most = (steps + AP_WAVES - 1) / AP_WAVES;
    if (!most) most = 1;
    ap_part w = {};
    w.most = (uint32_t)most;
    w.parts = w.most + a->c.n_seq;
    const uint64_t heads = (uint64_t)w.parts * a->n_heads;
    uint64_t n = 0;
    auto take = [&](uint64_t words) { const uint64_t o = n; n += (words + 3) / 4 * 4; return at + 4 * o; };
    w.acc = (float *)take(heads * a->c.hd);
    w.m = (float *)take(heads);
    w.l = (float *)take(heads);
    if (a->weight_out) w.score = (float *)take(rows * cap);     // by the table: the lengths are on the device
    if (a->c.n_seq > 64) w.plan = (uint32_t *)take((uint64_t)a->c.n_seq + 2 + w.parts);
    *bytes = 4 * n;
    return w;
}
extern "C" uint64_t sgk_attn_paged_scratch(const sgk_attn_paged_args *a) {
    uint64_t bytes;
    ap_plan(a, NULL, &bytes);
    return bytes;
}
extern "C" hipError_t sgk_attn_paged(const sgk_attn_paged_args *a, void *scratch, hipStream_t s, hipEvent_t done) {
    uint64_t bytes;
    const ap_part w = ap_plan(a, (char *)scratch, &bytes);
    const uint32_t hd = a->c.hd, grp = a->n_heads / a->c.n_kv;
    const int al = !((uintptr_t)a->q & 15) && a->q_stride % 4 == 0;
    const uint32_t ql = 3 * (hd / 32) * 1024, ol = AP_WAVES * (128 + grp * (hd + 4) * 4), lds = ql > ol ? ql : ol;
    if (w.plan) launch(k_attn_paged_plan, dim3(1), 1024, s, (hipEvent_t)NULL, *a, w);
    const dim3 grid(a->c.n_kv, w.parts);
    void (*const k)(sgk_attn_paged_args, ap_part, int) = hd == 64 ? k_attn_paged<64> : hd == 128 ? k_attn_paged<128> : k_attn_paged<256>;
    if (lds > 65536) {      // 16 heads of 256
        const hipError_t e = hipFuncSetAttribute((const void *)k, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    launch_lds(k, grid, AP_WAVES * 64, lds, s, (hipEvent_t)NULL, *a, w, al);
    uint32_t more = 0;      // workgroups a kv head for the weights: about 1024 in all, or 16 (16 x 4 heads: 16 9.8 us, 64 11.7; 8 heads: 16 10.8, 64 6.4)
    if (a->weight_out) {
        const uint64_t need = (((uint64_t)a->c.width << a->c.log) + TPB - 1) / TPB;
        const uint32_t most = max(16u, 1024u / (a->c.n_seq * a->c.n_kv));
        more = (uint32_t)(need < most ? need : most);
    }
    // a workgroup's dims of a head: all of them where sequences have few parts (16 x 2049 slots 54.9 -> 53 us, 262000 of one 186 -> 190)
    const uint32_t lanes = w.most <= 16 * a->c.n_seq ? hd / 4 : 16;
    void (*const join)(sgk_attn_paged_args, ap_part) = lanes == 16 ? k_attn_paged_join<16> : lanes == 32 ? k_attn_paged_join<32> : k_attn_paged_join<64>;
    launch(join, dim3(a->n_heads * (hd / (4 * lanes)) + more * a->c.n_kv, a->c.n_seq), TPB, s, done, *a, w);
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Eviction. The order of a (sequence, kv head)'s slots: recent ones first, then
// by weight, then the lower slot; the first `keep` stay. A workgroup holds the
// slots' keys in LDS (EV_HELD of them; past that it reads weight and pos again
// each time) and finds the keep-th by histograms of 11, 11 and 10 bits (weights
// share few exponents: with 8 bits the additions wait for each other), the last
// two over the keys of the first one's bin alone where those can be listed. Slots
// below keep that go are freed places, kept ones from keep on are moved rows: as
// many, both in rising order, so one prefix sum over both marks numbers them. No
// row that is read is written, so the moves need no order.
//
// A few rows too many (a cache that is held at keep) go one by one, the lowest of
// the workgroup's lowest. Long rows, where they are few, have several workgroups
// (below). Bound by the chain of passes of a CU over its keys, each some trips to
// LDS long, then by the moves: 64 rows of 2049 slots to 2048 5.9 us, 8 of 32768 to
// 4096 8 + 6.4 + 6.6 us in three launches (31.3 by one workgroup a row), and 15 to 16
// for the moves (59 MB, behind two dependent trips).
//
// The form follows the table, whose slots the host knows, not the lengths: one row out
// of a wider table pays for the launches that the table could need. 16 x 2049 to 2048,
// us a call: 14.7 in 2080 slots, 18.3 in 2128, 19.9 in 4096 to 32768, 23.5 in 65536;
// 2 x 4097 to 4096 14.7 in 4128, 26.4 in 32832. And more than EV_HELD slots that are
// held tight stay with one workgroup a row, which reads the keys again on every pass:
// 2 x 65537 to 65536 66 in as many slots, 32 in 131072.
//
// 256 threads a row are slower even at 4000 slots (23 us, 14). Loops are not unrolled
// far: code that runs once comes from memory (keys in registers, 64 a thread: 150 KB of
// it, 45 us).
// ---------------------------------------------------------------------------
#define EV_FEW 64u          // rows that the selecting workgroup moves itself (16 x 2080 slots to 2048: a call 19.1 us; with a launch for them 22.7)
#define EV_HELD 32896u      // keys in LDS: 32768 and a page of up to 128 more (one of 256 is past it)
#define EV_THREADS 1024
#define EV_BINS 2048u
#define EV_LIST 2048u       // keys of the first histogram's bin that are listed (as many as fit beside EV_HELD)
#define EV_PART 4096u       // slots of a workgroup where a row has several
#define EV_WIDE 24576u      // slots of a row from which on it has several (16000: 19.4 us and two more launches, 18.6 by one; 24000: 21.1, 24.1)
#define EV_OUT 8u           // rows too many that go one by one (2048 stay: 2 6.6 us, 11.3 by the border; 8 11.0, 11.6; 16 16.7, 11.8)
struct ev_list { uint32_t *hole, *mover, *n; };      // [row][most] twice, [row]: rows to move; NULL: the few are moved at once
__host__ __device__ static inline uint32_t ev_most(uint32_t keep, uint32_t cap) { return keep < cap - keep ? keep : cap - keep; }

// Rising with the order: 0xFFFFFFFF recent, 0 NaN. last: the largest position, so that last - pos does not wrap.
__device__ __forceinline__ uint32_t ev_key(float w, int32_t pos, int32_t last, uint32_t recent) {
    const uint32_t b = __float_as_uint(w + 0.0f);       // -0 as 0
    const uint32_t key = b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
    return (uint32_t)last - (uint32_t)pos < recent ? 0xFFFFFFFFu : w != w ? 0u : key;
}
// Row `from` to `to`: K and V by 16 bytes a thread, weight and pos with the first.
__device__ __forceinline__ void ev_move(const sgk_page_evict_args &a, uint32_t s, uint32_t h, uint32_t from, uint32_t to, uint32_t u, uint32_t units) {
    const uint64_t cap = (uint64_t)a.c.width << a.c.log, row = ((uint64_t)s * a.c.n_kv + h) * cap, wide = (uint64_t)a.c.n_kv * units;
    const int64_t x = page_row(a.c, s, from), y = page_row(a.c, s, to);
    if (u == 0) {
        a.weight_out[row + to] = a.weight[row + from];
        a.pos_out[row + to] = a.pos[row + from];
    }
    if (x < 0 || y < 0) return;
    const uint64_t xi = (uint64_t)x * wide + h * units + u, yi = (uint64_t)y * wide + h * units + u;
    const u16x8 kv = ((const u16x8 *)a.c.k)[xi], vv = ((const u16x8 *)a.c.v)[xi];
    ((u16x8 *)a.c.k)[yi] = kv;
    ((u16x8 *)a.c.v)[yi] = vv;
}
// Over the workgroup: the exclusive prefix sum of v, and the total. tmp: [2][16], halves taken in turn.
__device__ __forceinline__ uint32_t ev_scan(uint32_t v, uint32_t *total, uint32_t (*tmp)[16], int &at) {
    const uint32_t to = wave_scan(v), wv = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 63) tmp[at][wv] = to;
    __syncthreads();
    uint32_t before = to - v, all = 0;
#pragma unroll
    for (uint32_t i = 0; i < EV_THREADS / 64; i++) {
        const uint32_t x = tmp[at][i];
        if (i < wv) before += x;
        all += x;
    }
    at ^= 1;
    *total = all;
    return before;
}

template <bool HELD>
__global__ void __launch_bounds__(EV_THREADS) k_page_evict(sgk_page_evict_args a, ev_list w) {
    constexpr uint32_t T = EV_THREADS, W = T / 64, PER = EV_BINS / T;
    extern __shared__ uint32_t held[];
    __shared__ uint32_t bins[EV_BINS], tmp[2][16], marks[T], pick[4], list[EV_LIST];
    __shared__ int32_t lasts[W];
    __shared__ uint32_t few[2][EV_FEW], gone[EV_OUT];
    __shared__ uint64_t out[2][16];
    uint64_t dropped = 0;       // a bit a slot of the thread
    const uint32_t t = threadIdx.x, l = t & 63, wv = __builtin_amdgcn_readfirstlane(t >> 6), h = blockIdx.x, s = blockIdx.y;
    const uint32_t len = page_len(a.c, a.lens, s), cap = a.c.width << a.c.log, keep = min(a.keep, len);
    const uint64_t row = (uint64_t)s * a.c.n_kv + h;
    const float *wt = a.weight + row * cap;
    const int32_t *ps = a.pos + row * cap;
    float *wo = a.weight_out + row * cap;
    int32_t *po = a.pos_out + row * cap;
    if (t == 0 && w.n) w.n[row] = 0;
    // all of the first `keep` to the outputs; moved rows come over them, behind a barrier or a launch
    const bool cw = wo != wt, cp = po != ps;
    if (len <= a.keep) {
        if (cw) for (uint32_t j = t; j < keep; j += T) wo[j] = wt[j];
        if (cp) for (uint32_t j = t; j < keep; j += T) po[j] = ps[j];
        return;
    }
    for (uint32_t i = t; i < EV_BINS; i += T) bins[i] = 0;
    // eight of a thread's slots under way, the last one in place of those behind it
    int32_t last = INT32_MIN;
    for (uint32_t j0 = t; j0 - t < len; j0 += 8 * T) {
        int32_t p[8];
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) p[i] = ps[min(j0 + i * T, len - 1)];
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) {
            const uint32_t j = j0 + i * T;
            last = max(last, p[i]);
            if (HELD && j < len) held[j] = (uint32_t)p[i];
            if (cp && j < keep) po[j] = p[i];
        }
    }
    last = (int32_t)(wave_umax((uint32_t)last ^ 0x80000000u) ^ 0x80000000u);
    if (l == 0) lasts[wv] = last;
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < W; i++) last = max(last, lasts[i]);
    for (uint32_t j0 = t; j0 - t < len && (HELD || (cw && j0 - t < keep)); j0 += 8 * T) {
        float y[8];
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) y[i] = wt[min(j0 + i * T, len - 1)];
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) {
            const uint32_t j = j0 + i * T;
            if (HELD && j < len) held[j] = ev_key(y[i], (int32_t)held[j], last, a.recent);      // a thread's own
            if (cw && j < keep) wo[j] = y[i];
        }
    }
    __syncthreads();
    auto key_of = [&](uint32_t j) { return HELD ? held[j] : ev_key(wt[j], ps[j], last, a.recent); };
    uint32_t moves = 0;
    uint32_t *const holes = w.n ? w.hole + row * ev_most(a.keep, cap) : few[0], *const movers = w.n ? w.mover + row * ev_most(a.keep, cap) : few[1];
    if (HELD && len - keep <= EV_OUT) {
        // few rows too many, as in a cache that is held at `keep`: the lowest one (of alike keys the highest slot) out at a
        // time. A thread has the lowest of its slots in hand and looks again only when that one went.
        auto lowest = [&]() {
            uint64_t m = ~0ull;
            for (uint32_t j = t; j < len; j += T) m = min(m, (uint64_t)held[j] << 32 | (uint32_t)~j);
            return m;
        };
        uint64_t mine = lowest();
        for (uint32_t i = 0; i < len - keep; i++) {
            uint64_t m = row_min(mine);
            m = min(m, both<swap16>(m));
            m = min(m, both<swap32>(m));
            if (l == 0) out[i & 1][wv] = m;
            __syncthreads();
            const uint32_t j = ~(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)row_min(out[i & 1][l & 15]));
            if (t == 0) gone[i] = j;
            if (j % T == t) {               // its own slot, in no other thread's hands
                dropped |= 1ull << j / T;
                mine = ~0ull;
                for (uint32_t x = t; x < len; x += T)
                    if (!(dropped >> x / T & 1)) mine = min(mine, (uint64_t)held[x] << 32 | (uint32_t)~x);
            }
        }
        __syncthreads();
        // their places below keep in rising order, and the slots from keep on that stay
        if (t < 64) {
            const uint32_t n = len - keep, g = t < n ? gone[t] : UINT32_MAX, x = keep + t;
            uint32_t below = 0;
            bool stays = t < n;
            for (uint32_t i = 0; i < n; i++) {
                const uint32_t o = gone[i];
                below += o < g;
                stays = stays && o != x;
            }
            if (g < keep) holes[below] = g;
            const uint64_t m = __builtin_amdgcn_ballot_w64(stays);
            if (stays) movers[lanes_below(m)] = x;
            if (t == 0) pick[0] = (uint32_t)__popcll(m);
        }
        __syncthreads();
        moves = pick[0];
    } else {
    const uint32_t spans = (len + 63) / 64;
    // the keep-th key: `left` of the `here` keys with the border's upper bits stay
    uint32_t border = 0, left = keep, here = len, listed = UINT32_MAX;
    int at = 0;
    for (int pass = 0; pass < 3 && left != here; pass++) {
        const uint32_t shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, mask = pass == 2 ? 1023u : 2047u, up = pass == 0 ? 31 : pass == 1 ? 21 : 10;
        if (pass) {
            for (uint32_t i = t; i < EV_BINS; i += T) bins[i] = 0;
            __syncthreads();
        }
        if (pass == 0) {
            for (uint32_t j0 = t; j0 - t < len; j0 += 8 * T) {
                uint32_t key[8];
#pragma unroll
                for (uint32_t i = 0; i < 8; i++) key[i] = key_of(min(j0 + i * T, len - 1));
#pragma unroll
                for (uint32_t i = 0; i < 8; i++)
                    if (j0 + i * T < len) atomicAdd(&bins[key[i] >> 21], 1u);
            }
        } else if (listed <= EV_LIST) {
            for (uint32_t i = t; i < listed; i += T)
                if ((list[i] ^ border) >> up == 0) atomicAdd(&bins[list[i] >> shift & mask], 1u);
        } else {
#pragma unroll 8
            for (uint32_t j = t; j < len; j += T) {
                const uint32_t key = key_of(j);
                if ((key ^ border) >> up == 0) atomicAdd(&bins[key >> shift & mask], 1u);
            }
        }
        __syncthreads();
        // from the top: the bin in which `left` keys are reached
        uint32_t v[PER], sum = 0, unused;
#pragma unroll
        for (uint32_t i = 0; i < PER; i++) {
            v[i] = bins[EV_BINS - 1 - (t * PER + i)];
            sum += v[i];
        }
        uint32_t above = ev_scan(sum, &unused, tmp, at);
#pragma unroll
        for (uint32_t i = 0; i < PER; i++) {
            if (above < left && above + v[i] >= left) {
                pick[0] = EV_BINS - 1 - (t * PER + i);
                pick[1] = above;
                pick[2] = v[i];
            }
            above += v[i];
        }
        __syncthreads();
        border |= pick[0] << shift;
        left -= pick[1];
        here = pick[2];
        if (pass == 0 && left != here && here <= EV_LIST) {         // the other passes over that bin's keys alone
            listed = here;
            if (t == 0) pick[3] = 0;
            __syncthreads();
            for (uint32_t j0 = t; j0 - t < len; j0 += 8 * T) {
                uint32_t key[8];
#pragma unroll
                for (uint32_t i = 0; i < 8; i++) key[i] = key_of(min(j0 + i * T, len - 1));
#pragma unroll
                for (uint32_t i = 0; i < 8; i++)
                    if (key[i] >> 21 == border >> 21 && j0 + i * T < len) list[atomicAdd(&pick[3], 1u)] = key[i];
            }
        }
    }
    // Keys above the border stay and all of its own, or its own up to slot `tie`. A pass that was not needed left
    // lower bits 0.
    uint32_t tie = UINT32_MAX;
    if (left != here) {
        uint32_t seen = 0;
        for (uint32_t i0 = 0; i0 < spans; i0 += T) {
            for (uint32_t i = i0 + wv; i < min(i0 + T, spans); i += W) {
                const uint32_t j = i * 64 + l;
                const uint64_t m = __builtin_amdgcn_ballot_w64(j < len && key_of(min(j, len - 1)) == border);
                if (l == 0) marks[i - i0] = (uint32_t)__popcll(m);
            }
            __syncthreads();
            const uint32_t v = i0 + t < spans ? marks[t] : 0;
            uint32_t all;
            const uint32_t before = seen + ev_scan(v, &all, tmp, at);
            if (before < left && before + v >= left) { pick[0] = i0 + t; pick[1] = before; }
            seen += all;
            __syncthreads();
            if (seen >= left) break;
        }
        const uint32_t j = pick[0] * 64 + l;
        const bool mine = j < len && key_of(min(j, len - 1)) == border;
        const uint64_t m = __builtin_amdgcn_ballot_w64(mine);
        tie = pick[0] * 64 + (uint32_t)__builtin_ctzll(__builtin_amdgcn_ballot_w64(mine && pick[1] + lanes_below(m) + 1 == left));
    }
    // of four 64s of slots from i0 on, which of a lane's are freed (below keep) or moved (from keep on)
    auto marked = [&](uint32_t i0, bool (&m)[4]) {
        uint32_t key[4];
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) key[i] = key_of(min((i0 + i) * 64 + l, len - 1));
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) {
            const uint32_t j = (i0 + i) * 64 + l;
            const bool stays = tie == UINT32_MAX ? key[i] >= border : key[i] > border || (key[i] == border && j <= tie);
            m[i] = j < len && (j < keep) != stays;
        }
    };
    // The marks of each 64 slots, T of those at a time, and their prefix sums. A lane's marks are the bits of `mine`.
    uint64_t mine = 0;
    static_assert(T / W <= 64, "a bit for each 64 slots of a wave");
    auto count = [&](uint32_t s0) {
        mine = 0;
        uint32_t at = 0;
        for (uint32_t i0 = s0 + 4 * wv; i0 < min(s0 + T, spans); i0 += 4 * W, at += 4) {
            bool m[4];
            marked(i0, m);
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) {
                const uint64_t b = __builtin_amdgcn_ballot_w64(m[i]);
                if (l == 0) marks[i0 + i - s0] = (uint32_t)__popcll(b);
            }
            mine |= (uint64_t)(m[0] | m[1] << 1 | m[2] << 2 | m[3] << 3) << at;
        }
        __syncthreads();
    };
    uint32_t seen = 0;
    auto number = [&](uint32_t s0) {
        uint32_t all;
        const uint32_t before = seen + ev_scan(s0 + t < spans ? marks[t] : 0, &all, tmp, at);
        __syncthreads();
        marks[t] = before;
        seen += all;
        __syncthreads();
    };
    if (spans <= T) {
        __syncthreads();
        count(0);
        number(0);
        moves = seen / 2;
    } else {                    // all marks' number comes first
        for (uint32_t s0 = 0; s0 < spans; s0 += T) {
            __syncthreads();
            count(s0);
            number(s0);
        }
        moves = seen / 2;
        seen = 0;
    }
    for (uint32_t s0 = 0; s0 < spans; s0 += T) {
        if (spans > T) {
            __syncthreads();
            count(s0);
            number(s0);
        }
        uint32_t at = 0;
        for (uint32_t i0 = s0 + 4 * wv; i0 < min(s0 + T, spans); i0 += 4 * W, at += 4) {
            const uint32_t four = (uint32_t)(mine >> at) & 15;
            if (!__builtin_amdgcn_ballot_w64(four != 0)) continue;
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) {
                const uint32_t j = (i0 + i) * 64 + l, r = marks[i0 + i - s0] + lanes_below(__builtin_amdgcn_ballot_w64(four >> i & 1));
                if (four >> i & 1) *(j < keep ? holes + r : movers + (r - moves)) = j;
            }
        }
    }
    }
    if (w.n) {
        if (t == 0) w.n[row] = moves;
        return;
    }
    __syncthreads();
    const uint32_t units = a.c.hd / 8;
    for (uint32_t i = t; i < moves * units; i += T) ev_move(a, s, h, few[1][i / units], few[0][i / units], i % units, units);
}
// The same over several workgroups a row, EV_PART slots each, in three launches: the histograms of the parts (1); the border
// bin, the parts' marks that it decides, its keys listed in the order of their slots (2); the border and the marks (3). What a
// part's marks are numbered from follows from the counts of the parts before it and the list, so that no launch waits within.
struct ev_wide {
    uint32_t *hist, *count, *found;     // [row][parts][EV_BINS], [row][parts][2]: freed and moved, [row][4]: last, bin, left, here
    uint64_t *list;                     // [row][cap]: key, slot
    uint32_t parts;
};
struct ev_part {
    uint32_t len, keep, j0, used;       // used: parts with slots
    uint64_t row, cap;
    bool whole;                         // all slots stay
};
__device__ __forceinline__ ev_part ev_part_of(const sgk_page_evict_args &a) {
    ev_part p;
    p.len = page_len(a.c, a.lens, blockIdx.z);
    p.cap = (uint64_t)a.c.width << a.c.log;
    p.whole = p.len <= a.keep;
    p.keep = min(a.keep, p.len);
    p.j0 = blockIdx.x * EV_PART;
    p.used = (p.len + EV_PART - 1) / EV_PART;
    p.row = (uint64_t)blockIdx.z * a.c.n_kv + blockIdx.y;
    return p;
}
constexpr uint32_t EV_OWN = EV_PART / EV_THREADS;
__device__ __forceinline__ void ev_own(const sgk_page_evict_args &a, const ev_part &p, int32_t last, uint32_t (&key)[EV_OWN]) {
    float y[EV_OWN];
    int32_t x[EV_OWN];
#pragma unroll
    for (uint32_t i = 0; i < EV_OWN; i++) {
        const uint32_t j = min(p.j0 + i * EV_THREADS + threadIdx.x, p.len - 1);
        y[i] = a.weight[p.row * p.cap + j];
        x[i] = a.pos[p.row * p.cap + j];
    }
#pragma unroll
    for (uint32_t i = 0; i < EV_OWN; i++) key[i] = ev_key(y[i], x[i], last, a.recent);
}
// The numbers, in the order of the slots, of a part's marked slots.
__device__ __forceinline__ void ev_number(const bool (&m)[EV_OWN], uint32_t (&at)[EV_OWN], uint32_t *sub) {
    static_assert(EV_OWN * (EV_THREADS / 64) == 64, "a lane each");
    const uint32_t t = threadIdx.x, l = t & 63, wv = t >> 6;
    uint64_t b[EV_OWN];
#pragma unroll
    for (uint32_t i = 0; i < EV_OWN; i++) {
        b[i] = __builtin_amdgcn_ballot_w64(m[i]);
        if (l == 0) sub[i * (EV_THREADS / 64) + wv] = (uint32_t)__popcll(b[i]);
    }
    __syncthreads();
    const uint32_t v = sub[l], before = wave_scan(v) - v;
#pragma unroll
    for (uint32_t i = 0; i < EV_OWN; i++)
        at[i] = (uint32_t)__builtin_amdgcn_readlane((int)before, i * (EV_THREADS / 64) + __builtin_amdgcn_readfirstlane((int)wv)) + lanes_below(b[i]);
}
// Over the workgroup, two sums.
__device__ __forceinline__ void ev_sums(uint32_t &x, uint32_t &y, uint32_t (*tmp)[16]) {
    x = wave_sum(x);
    y = wave_sum(y);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) { tmp[0][threadIdx.x >> 6] = x; tmp[1][threadIdx.x >> 6] = y; }
    __syncthreads();
    x = y = 0;
#pragma unroll
    for (uint32_t i = 0; i < EV_THREADS / 64; i++) { x += tmp[0][i]; y += tmp[1][i]; }
    __syncthreads();
}
// The bin in which `left` keys from the top are reached, for all threads: bin, keys above it, its own. v: thread t's two bins,
// EV_BINS - 1 - 2 t and the one below.
__device__ __forceinline__ void ev_find(uint32_t left, uint32_t v0, uint32_t v1, uint32_t *pick, uint32_t (*tmp)[16], int &at) {
    static_assert(EV_BINS == 2 * EV_THREADS, "two bins a thread");
    uint32_t unused;
    const uint32_t b = EV_BINS - 1 - 2 * threadIdx.x, above = ev_scan(v0 + v1, &unused, tmp, at);
    if (above < left && above + v0 >= left) { pick[0] = b; pick[1] = above; pick[2] = v0; }
    else if (above + v0 < left && above + v0 + v1 >= left) { pick[0] = b - 1; pick[1] = above + v0; pick[2] = v1; }
    __syncthreads();
}
__global__ void __launch_bounds__(EV_THREADS) k_page_evict_hist(sgk_page_evict_args a, ev_list w, ev_wide v) {
    constexpr uint32_t T = EV_THREADS, W = T / 64;
    __shared__ uint32_t bins[EV_BINS];
    __shared__ int32_t lasts[W];
    const uint32_t t = threadIdx.x;
    const ev_part p = ev_part_of(a);
    const float *wt = a.weight + p.row * p.cap;
    const int32_t *ps = a.pos + p.row * p.cap;
    float *wo = a.weight_out + p.row * p.cap;
    int32_t *po = a.pos_out + p.row * p.cap;
    if (blockIdx.x == 0 && t == 0) w.n[p.row] = 0;
    // all of the first `keep` to the outputs; moved rows come over them in a later launch
#pragma unroll
    for (uint32_t i = 0; i < EV_OWN; i++) {
        const uint32_t j = p.j0 + i * T + t;
        if (j < p.keep && wo != wt) wo[j] = wt[j];
        if (j < p.keep && po != ps) po[j] = ps[j];
    }
    if (p.whole || p.j0 >= p.len) return;
    for (uint32_t i = t; i < EV_BINS; i += T) bins[i] = 0;
    int32_t last = INT32_MIN;
    for (uint32_t j0 = t; j0 - t < p.len; j0 += 16 * T) {
        int32_t x[16];
#pragma unroll
        for (uint32_t i = 0; i < 16; i++) x[i] = ps[min(j0 + i * T, p.len - 1)];
#pragma unroll
        for (uint32_t i = 0; i < 16; i++) last = max(last, x[i]);
    }
    last = (int32_t)(wave_umax((uint32_t)last ^ 0x80000000u) ^ 0x80000000u);
    if ((t & 63) == 0) lasts[t >> 6] = last;
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < W; i++) last = max(last, lasts[i]);
    uint32_t key[EV_OWN];
    ev_own(a, p, last, key);
#pragma unroll
    for (uint32_t i = 0; i < EV_OWN; i++)
        if (p.j0 + i * T + t < p.len) atomicAdd(&bins[key[i] >> 21], 1u);
    __syncthreads();
    uint32_t *to = v.hist + (p.row * v.parts + blockIdx.x) * EV_BINS;
    for (uint32_t i = t; i < EV_BINS; i += T) to[i] = bins[i];
    if (blockIdx.x == 0 && t == 0) v.found[4 * p.row] = (uint32_t)last;
}
__global__ void __launch_bounds__(EV_THREADS) k_page_evict_list(sgk_page_evict_args a, ev_wide v) {
    constexpr uint32_t T = EV_THREADS;
    __shared__ uint32_t tmp[2][16], pick[3], sub[64];
    const uint32_t t = threadIdx.x;
    const ev_part p = ev_part_of(a);
    if (p.whole || p.j0 >= p.len) return;
    const int32_t last = (int32_t)v.found[4 * p.row];
    uint32_t key[EV_OWN];
    ev_own(a, p, last, key);
    const uint32_t *hist = v.hist + p.row * v.parts * EV_BINS;
    int at = 0;
    uint64_t two = 0;       // a pair of bins: their sums stay below 2^32
#pragma unroll 8
    for (uint32_t q = 0; q < p.used; q++) two += *(const uint64_t *)(hist + q * EV_BINS + EV_BINS - 2 - 2 * t);
    ev_find(p.keep, (uint32_t)(two >> 32), (uint32_t)two, pick, tmp, at);
    const uint32_t bin = pick[0], left = p.keep - pick[1], here = pick[2];
    if (blockIdx.x == 0 && t == 0) { v.found[4 * p.row + 1] = bin; v.found[4 * p.row + 2] = left; v.found[4 * p.row + 3] = here; }
    uint32_t freed = 0, moved = 0;
    bool in[EV_OWN];
#pragma unroll
    for (uint32_t i = 0; i < EV_OWN; i++) {
        const uint32_t j = p.j0 + i * T + t, x = key[i] >> 21;
        in[i] = left != here && j < p.len && x == bin;
        freed += j < p.keep && x < bin;
        moved += j >= p.keep && j < p.len && x + (left == here) > bin;     // all of the bin stay, or the list tells
    }
    ev_sums(freed, moved, tmp);
    if (t == 0) { v.count[2 * (p.row * v.parts + blockIdx.x)] = freed; v.count[2 * (p.row * v.parts + blockIdx.x) + 1] = moved; }
    if (left == here) return;
    uint32_t base = 0, to[EV_OWN];
    for (uint32_t q = t & 63; q < blockIdx.x; q += 64) base += hist[q * EV_BINS + bin];
    base = wave_sum(base);
    ev_number(in, to, sub);
#pragma unroll
    for (uint32_t i = 0; i < EV_OWN; i++)
        if (in[i]) v.list[p.row * p.cap + base + to[i]] = (uint64_t)key[i] << 32 | (p.j0 + i * T + t);
}
__global__ void __launch_bounds__(EV_THREADS) k_page_evict_mark(sgk_page_evict_args a, ev_list w, ev_wide v) {
    constexpr uint32_t T = EV_THREADS;
    __shared__ uint32_t bins[EV_BINS], tmp[2][16], pick[3], sub[64];
    const uint32_t t = threadIdx.x;
    const ev_part p = ev_part_of(a);
    if (p.whole || p.j0 >= p.len) return;
    const uint32_t *found = v.found + 4 * p.row;
    const uint32_t listed = found[3];
    uint32_t border = found[1] << 21, left = found[2], here = listed, tie = UINT32_MAX;
    const uint64_t *list = v.list + p.row * p.cap;
    const bool all = left == here;      // the whole border bin stays: there is no list
    uint32_t key[EV_OWN];
    ev_own(a, p, (int32_t)found[0], key);
    int at = 0;
    for (int pass = 1; pass < 3 && left != here; pass++) {
        const uint32_t shift = pass == 1 ? 10 : 0, mask = pass == 1 ? 2047u : 1023u, up = pass == 1 ? 21 : 10;
        for (uint32_t i = t; i < EV_BINS; i += T) bins[i] = 0;
        __syncthreads();
#pragma unroll 4
        for (uint32_t i = t; i < listed; i += T) {
            const uint32_t k = (uint32_t)(list[i] >> 32);
            if ((k ^ border) >> up == 0) atomicAdd(&bins[k >> shift & mask], 1u);
        }
        __syncthreads();
        ev_find(left, bins[EV_BINS - 1 - 2 * t], bins[EV_BINS - 2 - 2 * t], pick, tmp, at);
        border |= pick[0] << shift;
        left -= pick[1];
        here = pick[2];
        __syncthreads();
    }
    if (left != here) {     // alike ones: up to the left-th slot
        uint32_t seen = 0;
        for (uint32_t i0 = 0; i0 < listed && seen < left; i0 += T) {
            const uint64_t e = i0 + t < listed ? list[i0 + t] : 0;
            const uint32_t is = i0 + t < listed && (uint32_t)(e >> 32) == border;
            uint32_t n;
            const uint32_t before = seen + ev_scan(is, &n, tmp, at);
            if (is && before + 1 == left) pick[0] = (uint32_t)e;
            seen += n;
        }
        __syncthreads();
        tie = pick[0];
    }
    auto stays = [&](uint32_t k, uint32_t j) { return tie == UINT32_MAX ? k >= border : k > border || (k == border && j <= tie); };
    // marks in front of the part's, and all freed ones
    uint32_t front = 0, moves = 0;
    for (uint32_t q = t; q < p.used; q += T) {
        const uint32_t *n = v.count + 2 * (p.row * v.parts + q);
        moves += n[0];
        if (q < blockIdx.x) front += n[0] + n[1];
    }
    for (uint32_t i = t; i < listed && !all; i += T) {
        const uint32_t j = (uint32_t)list[i];
        const bool s = stays((uint32_t)(list[i] >> 32), j), m = (j < p.keep) != s;
        moves += j < p.keep && !s;
        front += m && j < p.j0;
    }
    ev_sums(front, moves, tmp);
    bool m[EV_OWN];
    uint32_t to[EV_OWN];
#pragma unroll
    for (uint32_t i = 0; i < EV_OWN; i++) {
        const uint32_t j = p.j0 + i * T + t;
        m[i] = j < p.len && (j < p.keep) != stays(key[i], j);
    }
    ev_number(m, to, sub);
    const uint64_t most = ev_most(a.keep, (uint32_t)p.cap);
#pragma unroll
    for (uint32_t i = 0; i < EV_OWN; i++) {
        const uint32_t j = p.j0 + i * T + t, r = front + to[i];
        if (m[i]) *(j < p.keep ? w.hole + p.row * most + r : w.mover + p.row * most + (r - moves)) = j;
    }
    if (blockIdx.x == 0 && t == 0) w.n[p.row] = moves;
}
__global__ void __launch_bounds__(TPB) k_page_evict_move(sgk_page_evict_args a, ev_list w) {
    const uint32_t h = blockIdx.y, s = blockIdx.z, units = a.c.hd / 8, most = ev_most(a.keep, a.c.width << a.c.log);
    const uint64_t row = (uint64_t)s * a.c.n_kv + h, n = (uint64_t)w.n[row] * units;
    for (uint64_t i = (uint64_t)blockIdx.x * TPB + threadIdx.x; i < n; i += (uint64_t)gridDim.x * TPB)
        ev_move(a, s, h, w.mover[row * most + i / units], w.hole[row * most + i / units], (uint32_t)(i % units), units);
}
// The parts of a row that are selected by as many workgroups; 0: one workgroup.
static uint32_t ev_parts(const sgk_page_evict_args *a) {
    const uint32_t cap = a->c.width << a->c.log, parts = (cap + EV_PART - 1) / EV_PART;
    if (ev_most(a->keep, cap) <= EV_FEW || cap < EV_WIDE) return 0;
    return (uint64_t)parts * a->c.n_seq * a->c.n_kv <= 3ull * sgk_device_cus() / 2 ? parts : 0;
}
static uint64_t ev_plan(const sgk_page_evict_args *a, char *at, ev_list *w, ev_wide *v) {
    const uint64_t rows = (uint64_t)a->c.n_seq * a->c.n_kv, cap = (uint64_t)a->c.width << a->c.log, most = ev_most(a->keep, (uint32_t)cap);
    uint64_t n = 0;
    auto take = [&](uint64_t words) { char *o = at + 4 * n; n += (words + 3) / 4 * 4; return o; };
    *w = (ev_list){};
    *v = (ev_wide){};
    if (most <= EV_FEW) return 0;
    w->hole = (uint32_t *)take(rows * most);
    w->mover = (uint32_t *)take(rows * most);
    w->n = (uint32_t *)take(rows);
    v->parts = ev_parts(a);
    if (!v->parts) return 4 * n;
    v->list = (uint64_t *)take(2 * rows * cap);
    v->hist = (uint32_t *)take(rows * v->parts * EV_BINS);
    v->count = (uint32_t *)take(2 * rows * v->parts);
    v->found = (uint32_t *)take(4 * rows);
    return 4 * n;
}
extern "C" uint64_t sgk_page_evict_scratch(const sgk_page_evict_args *a) {
    ev_list w;
    ev_wide v;
    return ev_plan(a, NULL, &w, &v);
}
extern "C" hipError_t sgk_page_evict(const sgk_page_evict_args *a, void *scratch, hipStream_t s, hipEvent_t done) {
    const uint32_t cap = a->c.width << a->c.log, most = ev_most(a->keep, cap), rows = a->c.n_seq * a->c.n_kv;
    ev_list w;
    ev_wide v;
    ev_plan(a, (char *)scratch, &w, &v);
    const bool few = !w.n;
    if (v.parts) {
        const dim3 grid(v.parts, a->c.n_kv, a->c.n_seq);
        launch(k_page_evict_hist, grid, EV_THREADS, s, (hipEvent_t)NULL, *a, w, v);
        launch(k_page_evict_list, grid, EV_THREADS, s, (hipEvent_t)NULL, *a, v);
        launch(k_page_evict_mark, grid, EV_THREADS, s, (hipEvent_t)NULL, *a, w, v);
    } else {
        const bool held = cap <= EV_HELD;
        void (*const k)(sgk_page_evict_args, ev_list) = held ? k_page_evict<true> : k_page_evict<false>;
        const uint32_t lds = held ? cap * 4 : 0;
        if (lds > 49152) {
            const hipError_t e = hipFuncSetAttribute((const void *)k, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
            if (e != hipSuccess) return e;
        }
        launch_lds(k, dim3(a->c.n_kv, a->c.n_seq), EV_THREADS, lds, s, few ? done : (hipEvent_t)NULL, *a, w);
    }
    if (!few) {     // a trip a thread, but about 8192 workgroups in all
        const uint64_t b = ((uint64_t)most * (a->c.hd / 8) + TPB - 1) / TPB, all = max(8u, 8192u / rows);
        launch(k_page_evict_move, dim3((uint32_t)(b < all ? b : all), a->c.n_kv, a->c.n_seq), TPB, s, done, *a, w);
    }
    return hipGetLastError();
}
