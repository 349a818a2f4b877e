// sample.hip - a token a row from logits under temperature, top-k, top-p and
// min-p, by a given random number. The launcher is declared in kernels.h; its
// host checks are in hip.c.
#include "devutil.h"
#include "kernels.h"

// ---------------------------------------------------------------------------
// An id's weight is exp((x - max) / temperature), in 64 bits. Sums of weights
// are integers in units of the row's whole sum / 2^60 or so (the largest weight /
// 2^54 where at most 128 ids stay): whatever order the additions come in, the sums,
// the kept ids and the token are the same.
//
// A row is SM_IDS ids a workgroup, four a thread, over the chip, in three launches
// that each need what all of the last one found, and a fourth where the
// probabilities are wanted (without them the row's last workgroup of the third
// goes on). A row's settings are known on the device alone, so each launch does
// for a row what its kind needs:
//   few    top_k of SM_FEW at most (greedy: 1), in a row of SM_MAXIMA waves at most.
//          The top_k-th largest of the waves' maxima (1) is a bound that at least
//          top_k ids reach, and hardly more: those are listed (2), ranked by
//          comparing all with all, and the token is found among them (3). Where
//          fewer waves than top_k have any id (a mask, a short vocabulary), all ids
//          are listed, or past SM_LIST those that one workgroup finds by a histogram
//          (3).
//   all    no top_k, no top_p: the parts' sums (2), then the part in which the
//          token lies finds it (3).
//   border a histogram of the logits' distance from the largest, counts and sums
//          (2), gives the bins in which top_k and top_p end; their ids are listed,
//          the sums of the ids above them taken (3), and the list searched for the
//          exact borders (3 or 4): all with all, or past SM_NEAR entries by digits.
// A list that does not fit leaves the row to one workgroup, which goes over it digit by
// digit: thousands of ids in a bin at a border (alike ones, as 16-bit logits about 10 or
// 20 are, or a border 40 temperatures down), or above a few row's bound where the
// largest lie together in a few waves. One row of 151936 takes 1.0 to 1.5 ms then (bf16
// logits of mean 20 and deviation 2, top_p 0.95: 1.4; the same in f32 39 us).
//
// The logits are read once from memory and then from the last cache; what bounds
// a call is the chain of launches, each a few trips to memory long. One row of
// 151936 ids, top_k 20 and top_p 0.8: 3.0 + 6.7 + 5.8 us, the call 26, of which
// 8.8 are any call's. 16 rows of all kinds 6.2 + 11.9 + 17.2 (42 to 49); 4 rows with
// top_p and probabilities 4.4 + 8.4 + 6.9 + 13.1 (42). Ranking a few row's list in
// the second launch's last workgroup: 12.4 + 2.0 us against 6.4 + 5.9, so it is
// left to the third.
// ---------------------------------------------------------------------------
#define SM_THREADS 512
#define SM_WAVES (SM_THREADS / 64)
#define SM_IDS (4 * SM_THREADS)
#define SM_PARTS 512u       // of a row, at most: its parts take several rounds of SM_IDS past that
#define SM_FEW 128u         // a call, one row of 151936: top_k 20 25.4 us, 33.0 as the third kind; 127 29.7, 33.1 (16 rows, 20: 31.6, 52.7)
// Waves of a row of few, 16 a lane. A call with top_k 20: 262144 ids 25.2 us, 262145 as the third kind 35.5, as few by loops over the
// maxima 69; a million 47.7, 197.
#define SM_MAXIMA 1024u
#define SM_WGS 1024u        // workgroups that a launch has about (16 rows of 151936, a call with settings of all kinds: 512 42.7 us, 1024 41.4, 2048 46.4)
#define SM_LIST 2048u
#define SM_RANKED 128u      // entries that are compared all with all
#define SM_NEAR 256u        // entries of a list that is searched by comparing all with all (about 100 of them: 2 us, by digits 5)
#define SM_BINS 2048u
#define SM_NONE 0xFFFFFFFFu

// What the first launch found of a row: the largest and the lowest key, the ids that may be chosen, the weights' sum roughly.
// Of a few row that has been listed: ok is whether it has any id. One whose ok is more has yet to be.
struct sm_all { uint32_t best, low, ok; float top, sum; };
// Where top_k and top_p end: the bin of top_k's last id (SM_BINS: no top_k), ids and units before that bin; the bins in
// which top_p may end (SM_BINS: no top_p) and the units before them; the first bin that is listed; all units.
struct sm_border { uint32_t kbin, kabove, plo, phi, first; uint64_t ksum, psum, whole; };

// A row's place in the scratch memory.
struct sm_row {
    uint32_t *wave, *low, *ok;          // [parts][SM_WAVES] largest keys, [parts] lowest, [parts] ids that may be chosen
    float *sum;                         // [parts] of weights relative to the part's largest, roughly: for the units' size
    uint64_t *kept, *list, *binsum;     // [parts] units that stay, [SM_LIST] key and ~id, [SM_BINS]
    uint32_t *bincnt, *listed, *arrived, *out;      // [SM_BINS], [1], [1], [1 + 2 SM_FEW] few: number, ids, probabilities
    struct sm_all *all;                 // what 1 found, by 2
    struct sm_border *border;           // what 3 found
};
struct sm_plan { uint32_t parts, rounds; uint64_t row_bytes; char *at; };

__device__ __forceinline__ sm_row sm_at(const sm_plan &p, uint32_t r) {
    char *c = p.at + r * p.row_bytes;
    sm_row w;
    auto take = [&](uint64_t bytes) { char *x = c; c += (bytes + 15) / 16 * 16; return x; };
    w.sum = (float *)take(4 * p.parts);
    w.kept = (uint64_t *)take(8 * p.parts);
    w.list = (uint64_t *)take(8 * SM_LIST);
    w.binsum = (uint64_t *)take(8 * SM_BINS);
    w.bincnt = (uint32_t *)take(4 * SM_BINS);
    w.wave = (uint32_t *)take(4 * p.parts * SM_WAVES);
    w.low = (uint32_t *)take(4 * p.parts);
    w.ok = (uint32_t *)take(4 * p.parts);
    w.listed = (uint32_t *)take(8);
    w.arrived = w.listed + 1;
    w.out = (uint32_t *)take(4 * (1 + 2 * SM_FEW));
    w.all = (sm_all *)take(sizeof(sm_all));
    w.border = (sm_border *)take(sizeof(sm_border));
    return w;
}
static uint64_t sm_row_bytes(uint64_t parts) {
    uint64_t n = 0;
    auto take = [&](uint64_t bytes) { n += (bytes + 15) / 16 * 16; };
    take(4 * parts); take(8 * parts); take(8 * SM_LIST); take(8 * SM_BINS); take(4 * SM_BINS);
    take(4 * parts * SM_WAVES); take(4 * parts); take(4 * parts); take(8); take(4 * (1 + 2 * SM_FEW)); take(sizeof(sm_all)); take(sizeof(sm_border));
    return n;
}

// Rising with x; 0 for what is never chosen (NaN, -inf).
__device__ __forceinline__ uint32_t sm_key(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);       // -0 as 0
    return x > -INFINITY ? (b & 0x80000000u ? ~b : b | 0x80000000u) : 0;
}
__device__ __forceinline__ float sm_value(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key); }
// exp(z), z <= 0: 2^k e^r, |r| <= ln 2 / 2, by the series to r^12 (the next term is below 2^-52 of it). ln 2 in two parts, the
// first with 21 bits free below it, so that k times it is exact.
__device__ __forceinline__ double sm_exp(double z) {
    z = fmax(z, -1100.0);                       // 0 in 64 bits; NaN too
    const double k = rint(z * 1.4426950408889634);
    const double r = fma(-k, 0x1.a39ef35793c76p-33, fma(-k, 0x1.62e42feep-1, z));
    double p = 1.0 / 479001600;
    const double c[12] = {1.0, 1.0, 1.0 / 2, 1.0 / 6, 1.0 / 24, 1.0 / 120, 1.0 / 720, 1.0 / 5040, 1.0 / 40320, 1.0 / 362880, 1.0 / 3628800, 1.0 / 39916800};
#pragma unroll
    for (int i = 11; i >= 0; i--) p = fma(p, r, c[i]);
    return __builtin_amdgcn_ldexp(p, (int)k);
}
__device__ __forceinline__ double sm_weight(float x, float top, double inv) {
    return x == top ? 1.0 : x > -INFINITY && top < INFINITY ? sm_exp(((double)x - (double)top) * inv) : 0.0;
}
__device__ __forceinline__ float sm_rough(float x, float top, double inv) {
    return x == top ? 1.0f : x > -INFINITY && top < INFINITY ? exp2f((float)(((double)x - (double)top) * inv) * 1.44269504f) : 0.0f;
}
__device__ __forceinline__ uint64_t sm_units(double w, double up) { return w > 0.0 ? max((uint64_t)1, (uint64_t)rint(w * up)) : 0; }
// Over the workgroup, with 64 bits a wave in tmp.
template <typename T>
__device__ __forceinline__ T sm_sum(T v, void *tmp) {
    T *const x = (T *)tmp, w = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) x[threadIdx.x >> 6] = w;
    __syncthreads();
    T r = 0;
#pragma unroll
    for (int i = 0; i < SM_WAVES; i++) r += x[i];
    return r;
}
template <typename T>
__device__ __forceinline__ T sm_scan(T v, T *total, void *tmp) {      // exclusive
    T *const x = (T *)tmp;
    const T to = wave_scan(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) x[threadIdx.x >> 6] = to;
    __syncthreads();
    T before = 0, all = 0;
#pragma unroll
    for (uint32_t i = 0; i < SM_WAVES; i++) {
        if (i < threadIdx.x >> 6) before += x[i];
        all += x[i];
    }
    *total = all;
    return before + to - v;
}

struct sm_set { float temp, top_p, min_p, u; uint32_t top_k; double inv; bool few; };
__device__ __forceinline__ sm_set sm_settings(const sgk_sample_args &a, const sm_plan &p, uint32_t r) {
    const scalar_u32 *set = (const scalar_u32 *)(uintptr_t)(a.settings + 4ull * r);
    sm_set s = {__uint_as_float(set[0]), __uint_as_float(set[2]), __uint_as_float(set[3]), ((const scalar_f32 *)(uintptr_t)a.u)[r], set[1]};
    s.u = s.u > 0.0f ? fminf(s.u, 0x1.fffffep-1f) : 0.0f;
    if (!(s.temp > 0.0f)) { s.temp = 1.0f; s.top_k = 1; }
    if (!(s.top_p < 1.0f)) s.top_p = 1.0f;
    if (!(s.min_p > 0.0f)) s.min_p = 0.0f;
    if (s.min_p > 1.0f) s.top_k = 1;        // no weight is: the largest alone stays, of alike ones the lowest id
    s.inv = 1.0 / (double)s.temp;
    s.few = s.top_k && s.top_k <= SM_FEW && s.top_k <= p.parts * SM_WAVES && p.parts * SM_WAVES <= SM_MAXIMA;
    return s;
}
// The logits of ids i to i + 3 (NaN behind the last).
__device__ __forceinline__ void sm_four(const sgk_sample_args &a, uint32_t r, uint64_t i, int al, float (&x)[4]) {
    const float *q = a.x + (uint64_t)r * a.vocab + i;
    if (al && i < a.vocab) {
        const f32x4 v = *(const f32x4 *)q;
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = v[e];
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = i + e < a.vocab ? q[e] : NAN;
    }
}
// Four ids of round m of a part: their first, and their logits.
__device__ __forceinline__ uint32_t sm_load(const sgk_sample_args &a, const sm_plan &p, uint32_t r, uint32_t part, uint32_t m, int al, float (&x)[4]) {
    const uint64_t i = ((uint64_t)part * p.rounds + m) * SM_IDS + 4 * threadIdx.x;
    sm_four(a, r, i, al, x);
    return (uint32_t)i;
}
__device__ __forceinline__ sm_all sm_read(const sm_row &w, const sm_plan &p, const sm_set &s, uint64_t *tmp) {
    const uint32_t t = threadIdx.x, wv = t >> 6;
    uint32_t mine = 0, ok = 0, low = 0xFFFFFFFFu;
    float sum = 0.0f;
    if (t < p.parts) {
#pragma unroll
        for (uint32_t i = 0; i < SM_WAVES; i++) mine = max(mine, w.wave[t * SM_WAVES + i]);
        ok = w.ok[t];
        low = w.low[t];
        sum = w.sum[t];
    }
    uint32_t *const red = (uint32_t *)tmp;      // [3][SM_WAVES], and doubles behind
    const uint32_t b = wave_umax(mine), lw = ~wave_umax(~low), n = wave_sum(ok);
    if ((t & 63) == 0) { red[wv] = b; red[SM_WAVES + wv] = lw; red[2 * SM_WAVES + wv] = n; }
    __syncthreads();
    sm_all r = {};
    r.low = 0xFFFFFFFFu;
#pragma unroll
    for (int i = 0; i < SM_WAVES; i++) { r.best = max(r.best, red[i]); r.low = min(r.low, red[SM_WAVES + i]); r.ok += red[2 * SM_WAVES + i]; }
    r.top = sm_value(r.best);
    r.sum = fmaxf(sm_sum(mine ? sum * sm_rough(sm_value(mine), r.top, s.inv) : 0.0f, tmp + 2 * SM_WAVES), 1.0f);
    return r;
}
__device__ __forceinline__ double sm_unit(float sum) { return ldexp(1.0, 60 - ilogbf(sum)); }

// ---- 1: the parts' maxima and sums
__global__ void __launch_bounds__(SM_THREADS) k_sample_parts(sgk_sample_args a, sm_plan p, int al) {
    __shared__ uint64_t tmp[SM_WAVES];
    __shared__ uint32_t red[2 * SM_WAVES];
    const uint32_t t = threadIdx.x, part = blockIdx.x, r = blockIdx.y;
    const sm_row w = sm_at(p, r);
    const sm_set s = sm_settings(a, p, r);
    uint32_t best = 0, low = 0xFFFFFFFFu, ok = 0;
    float x[4];
    for (uint32_t m = 0; m < p.rounds; m++) {
        sm_load(a, p, r, part, m, al, x);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const uint32_t key = sm_key(x[e]);
            best = max(best, key);
            low = min(low, key - 1);
            ok += key != 0;
        }
    }
    for (uint32_t i = part * SM_THREADS + t; i < SM_BINS && !s.few; i += p.parts * SM_THREADS) { w.bincnt[i] = 0; w.binsum[i] = 0; }
    if (part == 0 && t == 0) { *w.listed = *w.arrived = 0; w.out[0] = 0; }
    best = wave_umax(best);
    low = ~wave_umax(~low);
    if ((t & 63) == 0) { w.wave[part * SM_WAVES + (t >> 6)] = best; red[t >> 6] = best; red[SM_WAVES + (t >> 6)] = low; }
    ok = sm_sum(ok, tmp);
#pragma unroll
    for (int i = 0; i < SM_WAVES; i++) { best = max(best, red[i]); low = min(low, red[SM_WAVES + i]); }
    if (t == 0) { w.ok[part] = ok; w.low[part] = ok ? low + 1 : 0xFFFFFFFFu; }
    if (s.few) return;
    float sum = 0.0f;
    const float top = sm_value(best);
    for (uint32_t m = 0; m < p.rounds && best; m++) {
        if (p.rounds > 1) sm_load(a, p, r, part, m, al, x);
#pragma unroll
        for (int e = 0; e < 4; e++) sum += sm_rough(x[e], top, s.inv);
    }
    sum = sm_sum(sum, tmp);
    if (t == 0) w.sum[part] = sum;
}

// The bins of the third kind: by distance from the largest logit, a range in which top_p ends whatever the logits are
// (weights below exp(-40) of the largest do not add up to 2^-24 of it), or all of it if that is less.
__device__ __forceinline__ float sm_bin_scale(const sm_set &s, const sm_all &all) {
    const float span = fminf(fmaxf(40.0f * s.temp, 24.0f), all.top - sm_value(all.low));
    return span > 0.0f && span < INFINITY ? (float)(SM_BINS - 2) / span : 0.0f;
}
__device__ __forceinline__ uint32_t sm_bin(float x, float top, float scale) {
    return x == top ? 0 : (uint32_t)fminf((top - x) * scale, (float)(SM_BINS - 1));
}
// Appends the ids of a thread that `in` marks to the row's list.
__device__ __forceinline__ void sm_append(const sm_row &w, const float (&x)[4], uint32_t i, uint32_t in) {
    if (!__builtin_amdgcn_ballot_w64(in != 0)) return;
    const uint32_t n = __popc(in), to = wave_scan(n);
    uint32_t base = 0;
    if ((threadIdx.x & 63) == 63) base = atomicAdd(w.listed, to);
    base = (uint32_t)__builtin_amdgcn_readlane((int)base, 63) + to - n;
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (in >> e & 1) {
            if (base < SM_LIST) __hip_atomic_store(w.list + base, (uint64_t)sm_key(x[e]) << 32 | (uint32_t)~(i + e), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            base++;
        }
}

// ---- 2: the few listed, the parts' sums, or the histogram
__global__ void __launch_bounds__(SM_THREADS) k_sample_count(sgk_sample_args a, sm_plan p, int al) {
    __shared__ uint64_t tmp[3 * SM_WAVES], sums[SM_BINS];
    __shared__ uint32_t cnts[SM_BINS];
    const uint32_t t = threadIdx.x, l = t & 63, part = blockIdx.x, r = blockIdx.y;
    const sm_row w = sm_at(p, r);
    const sm_set s = sm_settings(a, p, r);
    float x[4];
    uint32_t i = sm_load(a, p, r, part, 0, al, x);
    if (s.few) {
        // a bound that at least top_k ids reach: the top_k-th of the waves' maxima, its upper bits (every wave by itself)
        const uint32_t n = p.parts * SM_WAVES;
        uint32_t bound = 0, best = 0, least = 0xFFFFFFFFu;
        constexpr uint32_t C = SM_MAXIMA / 64;
        uint32_t c[C];
#pragma unroll
        for (uint32_t j = 0; j < C; j++) c[j] = j * 64 + l < n ? w.wave[j * 64 + l] : 0;
#pragma unroll
        for (uint32_t j = 0; j < C; j++) {
            best = max(best, c[j]);
            if (c[j]) least = min(least, c[j]);
        }
        best = wave_umax(best);
        least = ~wave_umax(~least);
        const uint32_t differ = best ^ least, high = differ ? 31 - __builtin_clz(differ) : 0;
        uint32_t waves = 0;     // that have any id
#pragma unroll
        for (uint32_t j = 0; j < C; j++) waves += (uint32_t)__popcll(__builtin_amdgcn_ballot_w64(c[j] != 0));
        uint32_t have = waves;
        // 11 bits of it at least, and more until few more waves reach it than have to
        if (have >= s.top_k) {
            bound = least & ~((2u << high) - 1);
            for (int b = (int)high; b >= 0 && (b > (int)high - 11 || have > s.top_k + s.top_k / 8); b--) {
                uint32_t k = 0;
#pragma unroll
                for (uint32_t j = 0; j < C; j++) {
                    if (j % 4 == 0 && j * 64 >= n) break;
                    k += (uint32_t)__popcll(__builtin_amdgcn_ballot_w64(c[j] >= (bound | 1u << b)));
                }
                if (k >= s.top_k) { bound |= 1u << b; have = k; }
            }
        }
        // too few waves for a bound, or just as many of which the last has few ids and so may have set a low one; and room for
        // more ids in them than can be listed
        if (__builtin_expect(waves < s.top_k + (p.rounds == 1 && a.vocab % 256 - 1 < 63) && waves * p.rounds > SM_LIST / 256, 0)) {
            const sm_all all = sm_read(w, p, s, tmp);
            if (all.ok > SM_LIST) {
                if (part == 0 && t == 0) *w.all = all;
                return;
            }
        }
        if (part == 0 && t == 0) *w.all = (sm_all){best, 0, best != 0, sm_value(best), 1.0f};
        bound = max(bound, 1u);
        for (uint32_t m = 0; m < p.rounds; m++) {
            if (m) i = sm_load(a, p, r, part, m, al, x);
            uint32_t in = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) in |= (uint32_t)(sm_key(x[e]) >= bound) << e;
            sm_append(w, x, i, in);
        }
        return;
    }
    const sm_all all = sm_read(w, p, s, tmp);
    if (part == 0 && t == 0) *w.all = all;
    if (!all.ok) return;
    const double up = sm_unit(all.sum);
    if ((!s.top_k || s.top_k >= all.ok) && s.top_p == 1.0f) {
        uint64_t q = 0;
        for (uint32_t m = 0; m < p.rounds; m++) {
            if (m) sm_load(a, p, r, part, m, al, x);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const double y = sm_weight(x[e], all.top, s.inv);
                if (y >= (double)s.min_p || x[e] == all.top) q += sm_units(y, up);
            }
        }
        q = sm_sum(q, tmp);
        if (t == 0) w.kept[part] = q;
        return;
    }
    for (uint32_t j = t; j < SM_BINS; j += SM_THREADS) { cnts[j] = 0; sums[j] = 0; }
    __syncthreads();
    const float scale = sm_bin_scale(s, all);
    const bool k_on = s.top_k && s.top_k < all.ok, p_on = s.top_p < 1.0f;       // counts for top_k, sums for top_p
    for (uint32_t m = 0; m < p.rounds; m++) {
        if (m) sm_load(a, p, r, part, m, al, x);
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (x[e] > -INFINITY) {
                const uint32_t b = sm_bin(x[e], all.top, scale);
                if (k_on) atomicAdd(&cnts[b], 1u);
                if (p_on) atomicAdd((unsigned long long *)&sums[b], (unsigned long long)sm_units(sm_weight(x[e], all.top, s.inv), up));
            }
    }
    __syncthreads();
    for (uint32_t j = t; j < SM_BINS; j += SM_THREADS) {
        if (cnts[j]) atomicAdd(w.bincnt + j, cnts[j]);
        if (sums[j]) atomicAdd((unsigned long long *)w.binsum + j, (unsigned long long)sums[j]);
    }
}

// ---- a list of ids in LDS: order (key, then ~id: the larger comes first), units, bin with SM_LOW if the weight is below min_p
#define SM_LOW 0x80000000u
struct sm_list { uint64_t order[SM_LIST], unit[SM_LIST]; uint32_t bin[SM_LIST], n; uint64_t tmp[2][SM_WAVES], sums[6][64], ahead[SM_THREADS]; uint32_t cnt[SM_WAVES], rank[SM_THREADS]; };

// The search of a list, by the workgroup: what stays under top_k and top_p (the lowest order that does), and, where `token`,
// the units of what stays and the token among it. It takes up to six jobs, one loop over one piece of code, since code that runs
// once comes from memory: 0 top_k's last key; 1, of alike keys, its last id; 2 the units that top_k left; 3 top_p's last key; 4 its
// last id; 5 the token. A job puts its entries aside, and finds the largest key (or ~id) from which on their units (or their number)
// and `before` come to `want`, the lowest if none does: six bits a step, from the highest in which they differ, the next six bits'
// sums in LDS, which every wave adds up. want > before; entries of no units do not count where units do.
__device__ __forceinline__ uint64_t wave_least(uint64_t v) {
    v = row_min(v);
    v = min(v, both<swap16>(v));
    return min(v, both<swap32>(v));
}
struct sm_result { uint64_t border, whole; uint32_t id; };
__device__ __forceinline__ uint64_t sm_lane(uint64_t v, int x) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), x) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, x);
}
__device__ __forceinline__ sm_result sm_search(sm_list &s, const sm_set &set, const sm_all &all, const sm_border &b, double up, bool token) {
    const uint32_t t = threadIdx.x, l = t & 63, wv = t >> 6, n = s.n;
    const bool k_on = b.kbin < SM_BINS, p_on = b.plo < SM_BINS;
    sm_result r = {0, b.whole, SM_NONE};
    uint32_t value = 0;
    uint64_t before = 0, want = 0;
    const bool near = n <= SM_NEAR;
    if (near) {
        // a short list: each entry against all, by two or four threads: how many are above it, and their units in top_p's bins
        uint64_t *const inside = &s.sums[0][0];
        static_assert(sizeof(s.sums) / 8 >= SM_NEAR && SM_NEAR == SM_THREADS / 2, "the units' place");
        const uint32_t each = n <= SM_THREADS / 4 ? SM_THREADS / 4 : SM_THREADS / 2, share = SM_THREADS / each, j = t & (each - 1);
        const uint32_t part = ((n + share - 1) / share + 7) / 8 * 8, from = t / each * part;
        const bool first = t < each && j < n;
        const uint32_t y = first ? s.bin[t] & ~SM_LOW : 0;
        const uint64_t u = first ? s.unit[t] : 0;
        if (t < SM_NEAR) inside[t] = y >= b.plo && y <= b.phi ? u : 0;
        if (t >= n && t < SM_NEAR) s.order[t] = 0;
        const uint64_t earlier = __builtin_amdgcn_ballot_w64(first && y != b.kbin);        // in bins before top_k's
        if (l == 0) s.cnt[wv] = (uint32_t)__popcll(earlier);
        __syncthreads();
        const uint64_t o = j < n ? s.order[j] : ~0ull;
        uint32_t rank = 0;
        uint64_t ahead = 0;
        for (uint32_t i = from; i < from + part; i += 8) {
            uint64_t x[8], z[8];
#pragma unroll
            for (uint32_t e = 0; e < 8; e++) { x[e] = s.order[i + e]; z[e] = inside[i + e]; }
#pragma unroll
            for (uint32_t e = 0; e < 8; e++) { rank += x[e] > o; ahead += x[e] > o ? z[e] : 0; }
        }
        s.rank[t] = rank;
        s.ahead[t] = ahead;
        __syncthreads();
        for (uint32_t i = 1; i < share; i++) {
            rank += s.rank[(t + i * each) & (SM_THREADS - 1)];
            ahead += s.ahead[(t + i * each) & (SM_THREADS - 1)];
        }
        uint32_t before_k = b.kabove;
#pragma unroll
        for (int i = 0; i < SM_WAVES; i++) before_k -= s.cnt[i];
        const bool ks = first && (y != b.kbin || before_k + rank < set.top_k);      // listed bins are not past top_k's
        if (k_on && p_on) {
            const uint64_t sum = wave_sum(ks && y == b.kbin ? u : 0);
            if (l == 0) s.tmp[0][wv] = sum;
            __syncthreads();
            r.whole = b.ksum;
#pragma unroll
            for (int i = 0; i < SM_WAVES; i++) r.whole += s.tmp[0][i];
        }
        bool stays = ks;
        if (p_on) {
            const double limit = ceil((double)set.top_p * (double)r.whole);
            want = max(limit > 0.0 ? (uint64_t)limit : 0, b.psum + 1);
            stays = ks && u && y >= b.plo && y <= b.phi && b.psum + ahead < want;
        }
        uint64_t lowest = wave_least(stays ? o : ~0ull);
        if (l == 0) s.tmp[1][wv] = lowest;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < SM_WAVES; i++) lowest = min(lowest, s.tmp[1][i]);
        r.border = lowest;
        __syncthreads();
    }
    for (int job = near ? 5 : k_on ? 0 : 3; job < (token ? 6 : 5); job++) {
        if (job >= 2 && job < 5 && !p_on) continue;
        const bool low = job == 1 || job >= 4, units = job >= 3;
        uint32_t mask = 0, cnt = 0, lo = 0xFFFFFFFFu, hi = 0;
        uint64_t sum = 0;
#pragma unroll 1
        for (uint32_t j = t, bit = 1; j < n; j += SM_THREADS, bit <<= 1) {
            const uint64_t o = s.order[j], u = s.unit[j];
            const uint32_t x = s.bin[j], y = x & ~SM_LOW, k = (uint32_t)(o >> 32), v = low ? (uint32_t)o : k;
            bool in = job < 3 ? y == b.kbin : u && (job < 5 ? y >= b.plo && y <= b.phi : !(x & SM_LOW));
            in = in && (job < 2 || o >= r.border) && ((job != 1 && job != 4) || k == value);
            if (!in) continue;
            mask |= bit;
            cnt++;
            sum += u;
            lo = min(lo, v);
            hi = max(hi, v);
        }
        sum = wave_sum(sum);
        cnt = wave_sum(cnt);
        lo = ~wave_umax(~lo);
        hi = wave_umax(hi);
        if (l == 0) { s.tmp[0][wv] = sum; s.tmp[1][wv] = (uint64_t)lo << 32 | hi; s.cnt[wv] = cnt; }
        if (t < 6 * 64) s.sums[t / 64][t % 64] = 0;
        __syncthreads();
        // a wave's lanes 0 to 7 (and 8 to 15, ...) have the waves'
        const uint64_t lh = s.tmp[1][l % SM_WAVES];
        lo = ~wave_umax(~(uint32_t)(lh >> 32));
        hi = wave_umax((uint32_t)lh);
        cnt = wave_sum(l < SM_WAVES ? s.cnt[l] : 0);
        sum = wave_sum(l < SM_WAVES ? s.tmp[0][l] : 0);
        bool skip = false;
        if (job == 0) {
            before = 0;
            want = set.top_k - b.kabove;
            skip = cnt <= want;
            if (skip) job = 1;
        } else if (job == 2) {
            r.whole = b.ksum + sum;
            skip = true;
        } else if (job == 3) {
            const double limit = ceil((double)set.top_p * (double)r.whole);
            before = b.psum;
            want = max(limit > 0.0 ? (uint64_t)limit : 0, before + 1);
        } else if (job == 5) {
            r.whole = sum;
            before = 0;
            want = (uint64_t)((double)set.u * (double)sum) + 1;
        }
        if (!skip) {
            int top = lo < hi ? 32 - __builtin_clz(lo ^ hi) : 0;       // bits that are not known yet
            uint64_t above = 0, own = 0;
            uint32_t found = top < 32 ? hi >> top << top : 0;
            for (int level = 0;; level++) {
                const int shift = max(top - 6, 0);
#pragma unroll 1
                for (uint32_t j = t, m = mask; m; j += SM_THREADS, m >>= 1) {
                    const uint64_t o = s.order[j];
                    const uint32_t v = (low ? (uint32_t)o : (uint32_t)(o >> 32)) ^ found;
                    if ((m & 1) && (top == 32 || v >> top == 0))
                        atomicAdd((unsigned long long *)&s.sums[level][v >> shift], (unsigned long long)(units ? s.unit[j] : 1));
                }
                __syncthreads();
                // from the highest on: the first at which `want` is reached, or the last that has any
                const uint64_t mine = s.sums[level][63 - l], to = wave_scan(mine);
                const uint64_t has = __builtin_amdgcn_ballot_w64(mine != 0), hit = __builtin_amdgcn_ballot_w64(mine != 0 && before + above + to >= want);
                const int x = hit ? __builtin_ctzll(hit) : has ? 63 - __builtin_clzll(has) : 63;
                above += sm_lane(to - mine, x);
                own = sm_lane(mine, x);
                found |= (uint32_t)(63 - x) << shift;
                top = shift;
                if (!top) break;
            }
            if (job == 0) {
                value = found;
                r.border = (uint64_t)found << 32;
                if (above + own <= want) job = 1;       // all of that key
                before = above;
            } else if (job == 3) {
                // of that key's ids, as many as it takes: of alike weights, so one or all are known without job 4
                value = found;
                r.border = max(r.border, (uint64_t)found << 32);
                before += above;
                if (before + own <= want || own == sm_units(sm_weight(sm_value(found), all.top, set.inv), up)) job = 4;
            } else if (job == 5) {
                r.id = ~found;
            } else {
                r.border = max(r.border, (uint64_t)value << 32 | found);
            }
        }
        __syncthreads();        // the sums are cleared again
    }
    return r;
}
// The list from memory; all threads. False: it does not fit.
__device__ __forceinline__ bool sm_fetch(sm_list &s, const sm_row &w, const sm_set &set, const sm_all &all, double up, float scale) {
    const uint32_t t = threadIdx.x;
    const uint32_t n = __hip_atomic_load(w.listed, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (n > SM_LIST) return false;
#pragma unroll 1
    for (uint32_t j = t; j < n; j += SM_THREADS) {
        const uint64_t o = __hip_atomic_load(w.list + j, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const float x = sm_value((uint32_t)(o >> 32));
        const double y = sm_weight(x, all.top, set.inv);
        s.order[j] = o;
        s.unit[j] = sm_units(y, up);
        s.bin[j] = (set.few ? 0 : sm_bin(x, all.top, scale)) | (y >= (double)set.min_p || x == all.top ? 0 : SM_LOW);
    }
    if (t == 0) s.n = n;
    __syncthreads();
    return true;
}

// The token of a row's part in which the units pass `want` (counted from the part's start), and the part's probabilities.
template <typename Stays>
__device__ __forceinline__ void sm_pick(const sgk_sample_args &a, const sm_plan &p, uint32_t r, uint32_t part, int al, const sm_set &s, float top, double up,
                                        double whole, bool here, uint64_t want, uint64_t *tmp, uint32_t *least, Stays stays) {
    if (!here && !a.probs) return;
    uint64_t before = 0;
    if (threadIdx.x == 0) *least = SM_NONE;
    float next[4];
    uint32_t ni = sm_load(a, p, r, part, 0, al, next);
    for (uint32_t m = 0; m < p.rounds; m++) {
        float x[4], out[4];
        const uint32_t i = ni;
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = next[e];
        if (m + 1 < p.rounds) ni = sm_load(a, p, r, part, m + 1, al, next);
        uint64_t q[4], mine = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const double y = sm_weight(x[e], top, s.inv);
            const bool k = x[e] > -INFINITY && (y >= (double)s.min_p || x[e] == top) && stays(x[e], i + e);
            q[e] = k ? sm_units(y, up) : 0;
            out[e] = q[e] ? (float)(y * up / whole) : 0.0f;
            mine += q[e];
        }
        if (here) {
            uint64_t all, at = before + sm_scan(mine, &all, tmp);
            before += all;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                at += q[e];
                if (q[e] && at > want) { atomicMin(least, i + e); break; }
            }
        }
        if (a.probs && i < a.vocab) {
            float *d = a.probs + (uint64_t)r * a.vocab + i;
            if (al) *(f32x4 *)d = (f32x4){out[0], out[1], out[2], out[3]};
            else
                for (int e = 0; e < 4; e++) if (i + e < a.vocab) d[e] = out[e];
        }
    }
    if (!here) return;
    __syncthreads();
    if (threadIdx.x == 0) a.token[r] = *least;
}

// A row whose list does not fit: one workgroup, the borders of top_k and top_p by the digits of the keys, 8 bits a pass over the row.
__device__ __forceinline__ void sm_slow(const sgk_sample_args &a, uint32_t r, const sm_set &set, sm_list *room) {
    uint64_t *const hist = room->order, *const tmp = hist + 256, *const pick = tmp + SM_WAVES;
    uint32_t *const tmp32 = room->bin, &token = room->n;
    const uint32_t t = threadIdx.x, v = a.vocab, top_k = set.top_k;
    const float *x = a.x + (uint64_t)r * v, top_p = set.top_p, min_p = set.min_p, u = set.u;
    uint32_t best = 0, ok = 0;
    for (uint32_t i = t; i < v; i += SM_THREADS) {
        const uint32_t key = sm_key(x[i]);
        best = max(best, key);
        ok += key != 0;
    }
    for (int d = 1; d < 64; d <<= 1) best = max(best, (uint32_t)__shfl_xor(best, d));
    if ((t & 63) == 0) tmp32[t >> 6] = best;
    __syncthreads();
    for (int i = 0; i < (int)SM_WAVES; i++) best = max(best, tmp32[i]);
    __syncthreads();
    ok = sm_sum(ok, tmp32);
    float *probs = a.probs ? a.probs + (uint64_t)r * v : NULL;
    const float top = __uint_as_float(best & 0x80000000u ? best ^ 0x80000000u : ~best);
    const double inv = set.inv;
    // top-k: the last key that stays, and how many of its ids
    uint32_t border = 0, ties = SM_NONE;
    if (top_k && top_k < ok) {
        uint64_t left = top_k;
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (t < 256) hist[t] = 0;
            __syncthreads();
            for (uint32_t i = t; i < v; i += SM_THREADS) {
                const uint32_t key = sm_key(x[i]);
                if (key && (shift == 24 || key >> (shift + 8) == border >> (shift + 8))) atomicAdd((unsigned long long *)&hist[key >> shift & 255], 1ull);
            }
            __syncthreads();
            if (t == 0) {
                uint32_t b = 255;
                while (hist[b] < left) left -= hist[b--];
                pick[0] = border | b << shift;
                pick[1] = left;
            }
            __syncthreads();
            border = (uint32_t)pick[0];
            left = pick[1];
            __syncthreads();
        }
        ties = (uint32_t)left;
    }
    // the sum of what top-k left: first in floating point, for the unit, then in units
    double part = 0.0;
    for (uint32_t i = t; i < v; i += SM_THREADS) if (sm_key(x[i]) > border) part += sm_weight(x[i], top, inv);
    double sum = sm_sum(part, tmp);
    const float bx = __uint_as_float(border & 0x80000000u ? border ^ 0x80000000u : ~border);
    if (border) sum += ties * sm_weight(bx, top, inv);
    const double up = ldexp(1.0, 61 - ilogb(sum));
    uint64_t whole = 0;
    for (uint32_t i = t; i < v; i += SM_THREADS) if (sm_key(x[i]) > border) whole += sm_units(sm_weight(x[i], top, inv), up);
    whole = sm_sum(whole, tmp);
    if (border) whole += ties * sm_units(sm_weight(bx, top, inv), up);
    // top-p: the lowest key before which the sum is below p * whole
    if (top_p < 1.0f) {
        const double want = (double)top_p * (double)whole;
        uint64_t above = 0;
        uint32_t low = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (t < 256) hist[t] = 0;
            __syncthreads();
            for (uint32_t i = t; i < v; i += SM_THREADS) {
                const uint32_t key = sm_key(x[i]);
                if (key > border && (shift == 24 || key >> (shift + 8) == low >> (shift + 8)))
                    atomicAdd((unsigned long long *)&hist[key >> shift & 255], (unsigned long long)sm_units(sm_weight(x[i], top, inv), up));
            }
            __syncthreads();
            if (t == 0) {
                if (border && (shift == 24 || border >> (shift + 8) == low >> (shift + 8)))
                    hist[border >> shift & 255] += ties * sm_units(sm_weight(bx, top, inv), up);
                // the lowest digit with something in it before which the sum is below `want`; the highest if none is
                uint32_t at = 256;
                uint64_t sum_at = above, run = above;
                for (int b = 255; b >= 0; b--) {
                    if (!hist[b]) continue;
                    if (at < 256 && !((double)run < want)) break;
                    at = (uint32_t)b;
                    sum_at = run;
                    run += hist[b];
                }
                pick[0] = low | at << shift;
                pick[1] = sum_at;
            }
            __syncthreads();
            low = (uint32_t)pick[0];
            above = pick[1];
            __syncthreads();
        }
        const float lx = __uint_as_float(low & 0x80000000u ? low ^ 0x80000000u : ~low);
        const double each = (double)sm_units(sm_weight(lx, top, inv), up), n = ceil((want - (double)above) / each);
        const uint32_t most = low == border ? ties : SM_NONE;
        border = low;
        ties = n < 1.0 ? 1 : n < (double)most ? (uint32_t)n : most;
    }
    // what stays: keys above the border and the first ties of it, with a weight of min_p at least
    whole = 0;
    uint32_t seen = 0;
    if (t == 0) token = SM_NONE;
    for (int pass = 0; pass < 2; pass++) {
        const double over = (double)whole;
        const uint64_t want = (uint64_t)((double)u * over);
        uint64_t cum = 0;
        seen = 0;
        for (uint32_t i0 = 0; i0 < v; i0 += SM_THREADS) {
            const uint32_t i = i0 + t, key = i < v ? sm_key(x[i]) : 0;
            const bool tie = key && key == border;
            uint32_t n;
            const uint32_t rank = seen + sm_scan((uint32_t)tie, &n, tmp32);
            seen += n;
            const double w = key && (key > border || (tie && rank < ties)) ? sm_weight(x[i], top, inv) : 0.0;
            const uint64_t q = w >= (double)min_p || !(min_p > 0.0f) || key == best ? sm_units(w, up) : 0;
            if (!pass) { whole += q; continue; }
            uint64_t all;
            const uint64_t before = cum + sm_scan(q, &all, tmp);
            cum += all;
            if (q && before + q > want) atomicMin(&token, i);
            if (probs && i < v) probs[i] = q ? (float)(w * up / over) : 0.0f;
        }
        if (!pass) whole = sm_sum(whole, tmp);
    }
    __syncthreads();
    if (t == 0) a.token[r] = token;
}
// A few row whose waves give no bound and whose ids (all.ok) are too many: the ids of the waves that have any, down to the bin in
// which top_k ends, are listed. By one workgroup; `room` is used.
__device__ __forceinline__ void sm_narrow(const sgk_sample_args &a, const sm_plan &p, uint32_t r, const sm_row &w, int al, const sm_set &s, const sm_all &all,
                                          sm_list *room) {
    constexpr uint32_t PER = SM_BINS / SM_THREADS, A = 4;       // A of a wave's blocks of 256 ids under way
    static_assert(SM_BINS + SM_FEW + 1 <= 2 * SM_LIST, "room for the counts and the waves");
    uint32_t *const cnts = (uint32_t *)room->order, *const some = cnts + SM_BINS, *const last = some + SM_FEW;
    const uint32_t t = threadIdx.x, l = t & 63, waves = p.parts * SM_WAVES;
    const float scale = sm_bin_scale(s, all);
    for (uint32_t j = t; j < SM_BINS; j += SM_THREADS) cnts[j] = 0;
    uint32_t n = 0;         // waves that have any: top_k at most
    for (uint32_t j = l; j - l < waves; j += 64) {
        const bool has = j < waves && w.wave[j];
        const uint64_t any = __builtin_amdgcn_ballot_w64(has);
        if (has && t < 64 && n + lanes_below(any) < SM_FEW) some[n + lanes_below(any)] = j;
        n += (uint32_t)__popcll(any);
    }
    __syncthreads();
    const uint32_t blocks = min(n, SM_FEW) * p.rounds;
    auto each = [&](auto f) {
        for (uint32_t q0 = __builtin_amdgcn_readfirstlane(t >> 6); q0 < blocks; q0 += A * SM_WAVES) {
            float x[A][4];
            uint64_t i[A];
#pragma unroll
            for (uint32_t b = 0; b < A; b++) {
                const uint32_t q = q0 + b * SM_WAVES, v = q < blocks ? some[q / p.rounds] : 0;
                i[b] = q < blocks ? ((uint64_t)(v / SM_WAVES) * p.rounds + q % p.rounds) * SM_IDS + 4 * (v % SM_WAVES * 64 + l) : a.vocab;
                sm_four(a, r, i[b], al, x[b]);
            }
#pragma unroll
            for (uint32_t b = 0; b < A; b++) f(x[b], (uint32_t)i[b]);
        }
    };
    each([&](const float (&x)[4], uint32_t) {
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (x[e] > -INFINITY) atomicAdd(&cnts[sm_bin(x[e], all.top, scale)], 1u);
    });
    __syncthreads();
    uint32_t cnt[PER], c = 0, unused;
#pragma unroll
    for (uint32_t i = 0; i < PER; i++) {
        cnt[i] = cnts[t * PER + i];
        c += cnt[i];
    }
    c = sm_scan(c, &unused, room->tmp);
#pragma unroll
    for (uint32_t i = 0; i < PER; i++) {
        if (c < s.top_k && c + cnt[i] >= s.top_k) *last = t * PER + i;
        c += cnt[i];
    }
    __syncthreads();
    const uint32_t bin = *last;
    each([&](const float (&x)[4], uint32_t i) {
        uint32_t in = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) in |= (uint32_t)(x[e] > -INFINITY && sm_bin(x[e], all.top, scale) <= bin) << e;
        sm_append(w, x, i, in);
    });
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");        // what this wave wrote has arrived
    __syncthreads();
}
// ---- 3. LAST: the row's last workgroup goes on to the token, and no fourth launch follows; what it takes from the others
// has been written through to memory.
template <bool LAST>
__global__ void __launch_bounds__(SM_THREADS) k_sample_border(sgk_sample_args a, sm_plan p, int al) {
    __shared__ uint64_t tmp[SM_WAVES];
    __shared__ uint32_t least, tmp32[SM_WAVES];
    __shared__ sm_border found;
    __shared__ sm_list list;
    __shared__ struct { uint32_t rank[4][SM_RANKED]; uint64_t ahead[4][SM_RANKED]; } ranked;
    auto &ranks = ranked.rank;
    auto &aheads = ranked.ahead;
    const uint32_t t = threadIdx.x, part = blockIdx.x, r = blockIdx.y;
    const sm_row w = sm_at(p, r);
    const sm_set s = sm_settings(a, p, r);
    if (s.few && part) return;
    const sm_all all = *w.all;
    const uint32_t few_listed = s.few ? *w.listed : 0;      // with all, before anything waits for that
    if (!all.ok) {
        if (LAST && part == 0 && t == 0) a.token[r] = SM_NONE;
        return;
    }
    const bool k_on = s.top_k && s.top_k < all.ok, p_on = s.top_p < 1.0f, listed_kind = s.few || k_on || p_on;
    const double up = s.few ? 0x1p54 : sm_unit(all.sum);        // few: 2^7 ids at most
    const float scale = s.few ? 0.0f : sm_bin_scale(s, all);
    sm_border b;
    bool here = true;
    uint32_t mine_part = part;
    uint64_t want = 0, total = 0;
    if (s.few) {
        // not listed yet (32000 ids, top_k 126 of 125 waves: a call 44 us, 318 with all ids listed; 4096 in a row of a mask, top_k 18 of 17: 29, 950)
        uint32_t listed = few_listed;
        if (__builtin_expect(all.ok > 1, 0)) {
            sm_narrow(a, p, r, w, al, s, all, &list);
            listed = __hip_atomic_load(w.listed, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        if (listed <= SM_RANKED) {
            // each entry against all: four groups of waves take a quarter of the others each, for 64 or 128 entries
            const uint32_t l = t & 63, half = t >> 6 & 1, j = 64 * half + l, from = (t >> 7) * (SM_RANKED / 4);
            if (t < SM_RANKED) {
                const uint64_t o = t < listed ? w.list[t] : 0;
                const double y = t < listed ? sm_weight(sm_value((uint32_t)(o >> 32)), all.top, s.inv) : 0.0;
                list.order[t] = o;
                list.unit[t] = sm_units(y, up);
                list.bin[t] = t < listed && (y >= (double)s.min_p || sm_value((uint32_t)(o >> 32)) == all.top) ? 0 : SM_LOW;
            }
            __syncthreads();
            uint32_t rank = 0;
            uint64_t ahead = 0;
            if (64 * half < listed) {
                const uint64_t o = list.order[j];
                for (uint32_t i = from; i < min(from + SM_RANKED / 4, listed); i++)
                    if (list.order[i] > o) { rank++; ahead += list.unit[i]; }
            }
            ranks[t >> 7][j] = rank;
            aheads[t >> 7][j] = ahead;
            __syncthreads();
            if (t >= 64) return;
            // lane l has entries l and 64 + l
            uint64_t unit[2], before[2], kept = 0;
            uint32_t id[2];
            bool stays[2];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const uint32_t x = 64 * i + l, k = ranks[0][x] + ranks[1][x] + ranks[2][x] + ranks[3][x];
                before[i] = aheads[0][x] + aheads[1][x] + aheads[2][x] + aheads[3][x];
                unit[i] = list.unit[x];
                id[i] = ~(uint32_t)list.order[x];
                stays[i] = x < listed && k < s.top_k;
                kept += stays[i] ? unit[i] : 0;
            }
            if (s.top_p < 1.0f) {
                const double want = ceil((double)s.top_p * (double)wave_sum(kept));
                const uint64_t units = want > 1.0 ? (uint64_t)want : 1;
                stays[0] = stays[0] && before[0] < units;
                stays[1] = stays[1] && before[1] < units;
            }
            kept = 0;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                stays[i] = stays[i] && !(list.bin[64 * i + l] & SM_LOW);
                kept += stays[i] ? unit[i] : 0;
            }
            const uint64_t whole = wave_sum(kept), want = (uint64_t)((double)s.u * (double)whole);
            // the units of the ids up to an entry's own, over those that stay
            uint64_t upto[2] = {0, 0};
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                uint64_t left = __builtin_amdgcn_ballot_w64(stays[i]);
                if (a.probs && stays[i]) {
                    const uint32_t at = m + lanes_below(left);
                    w.out[1 + 2 * at] = id[i];
                    w.out[2 + 2 * at] = __float_as_uint((float)(sm_weight(sm_value((uint32_t)(list.order[64 * i + l] >> 32)), all.top, s.inv) * up / (double)whole));
                }
                m += (uint32_t)__popcll(left);
                for (; left; left &= left - 1) {
                    const int x = __builtin_ctzll(left);
                    const uint32_t d = (uint32_t)__builtin_amdgcn_readlane((int)id[i], x);
                    const uint64_t y = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(unit[i] >> 32), x) << 32 |
                                       (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)unit[i], x);
                    if (d <= id[0]) upto[0] += y;
                    if (d <= id[1]) upto[1] += y;
                }
            }
#pragma unroll
            for (int i = 0; i < 2; i++)
                if (stays[i] && unit[i] && upto[i] > want && upto[i] - unit[i] <= want) a.token[r] = id[i];
            if (t == 0) w.out[0] = m;
            return;
        }
        b = (sm_border){0, 0, s.top_p < 1.0f ? 0 : SM_BINS, 0, 0, 0, 0, 0};
    } else if (!k_on && !p_on) {
        const uint64_t mine = t < p.parts ? w.kept[t] : 0, before = sm_scan(mine, &total, tmp);
        want = (uint64_t)((double)s.u * (double)total);
        if (t == part) { found.ksum = before; found.psum = mine; }
        __syncthreads();
        here = want >= found.ksum && want < found.ksum + found.psum;
        want -= found.ksum;
    } else {
        // the bins in which top_k and top_p end
        constexpr uint32_t PER = SM_BINS / SM_THREADS;
        uint32_t cnt[PER], c = 0, nall;
        uint64_t sum[PER], u = 0, whole;
#pragma unroll
        for (uint32_t i = 0; i < PER; i++) {
            cnt[i] = w.bincnt[t * PER + i];
            sum[i] = w.binsum[t * PER + i];
            c += cnt[i];
            u += sum[i];
        }
        c = sm_scan(c, &nall, tmp32);
        u = sm_scan(u, &whole, tmp);
        if (t == 0) found = (sm_border){SM_BINS, 0, SM_BINS, SM_BINS, 0, 0, 0, whole};
        __syncthreads();
        uint64_t klo = whole, khi = whole;
        if (k_on) {
            uint32_t cc = c;
            uint64_t uu = u;
#pragma unroll
            for (uint32_t i = 0; i < PER; i++) {
                if (cc < s.top_k && cc + cnt[i] >= s.top_k) { found.kbin = t * PER + i; found.kabove = cc; found.ksum = uu; found.psum = uu + sum[i]; }
                cc += cnt[i];
                uu += sum[i];
            }
            __syncthreads();
            klo = found.ksum;
            khi = found.psum;
            __syncthreads();
        }
        if (p_on) {
            const double dlo = ceil((double)s.top_p * (double)klo), dhi = ceil((double)s.top_p * (double)khi);
            const uint64_t wlo = dlo > 1.0 ? (uint64_t)dlo : 1, whi = dhi > 1.0 ? (uint64_t)dhi : 1;
            uint64_t uu = u;
#pragma unroll
            for (uint32_t i = 0; i < PER; i++) {
                if (uu < wlo && uu + sum[i] >= wlo) { found.plo = t * PER + i; found.psum = uu; }
                if (uu < whi && uu + sum[i] >= whi) found.phi = t * PER + i;
                uu += sum[i];
            }
            __syncthreads();
        }
        b = found;
        if (p_on && b.kbin < SM_BINS) b.phi = min(b.phi, b.kbin);
        b.first = p_on ? b.plo : b.kbin;
        if (part == 0 && t == 0) *w.border = b;
        uint64_t q = 0;
        for (uint32_t m = 0; m < p.rounds; m++) {
            float x[4];
            const uint32_t i = sm_load(a, p, r, part, m, al, x);
            uint32_t in = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (!(x[e] > -INFINITY)) continue;
                const uint32_t y = sm_bin(x[e], all.top, scale);
                if (y < b.first) {
                    const double z = sm_weight(x[e], all.top, s.inv);
                    if (z >= (double)s.min_p || x[e] == all.top) q += sm_units(z, up);
                } else if (y == b.kbin || (p_on && y <= b.phi)) {
                    in |= 1u << e;
                }
            }
            sm_append(w, x, i, in);
        }
        q = sm_sum(q, tmp);
        if (t == 0) __hip_atomic_store(w.kept + part, q, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (!LAST) return;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");        // what this wave wrote has arrived
        __syncthreads();
        if (t == 0) least = __hip_atomic_fetch_add(w.arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if (least != p.parts - 1) return;
        __syncthreads();
    }
    sm_result f = {};
    if (listed_kind) {
        if (!sm_fetch(list, w, s, all, up, scale)) {
            if (LAST) sm_slow(a, r, s, &list);
            return;
        }
        f = sm_search(list, s, all, b, up, s.few);
    }
    auto in = [&](uint32_t j) { return list.order[j] >= f.border && !(list.bin[j] & SM_LOW); };
    if (s.few) {
        if (t == 0) a.token[r] = f.id;
        if (!a.probs || t >= 64) return;
        uint32_t n = 0;
        for (uint32_t j0 = 0; j0 < list.n; j0 += 64) {
            const uint32_t j = j0 + t;
            const bool k = j < list.n && in(j);
            const uint64_t m = __builtin_amdgcn_ballot_w64(k);
            const uint32_t at = n + lanes_below(m);
            if (k && at < SM_FEW) {
                w.out[1 + 2 * at] = ~(uint32_t)list.order[j];
                w.out[2 + 2 * at] = __float_as_uint((float)(sm_weight(sm_value((uint32_t)(list.order[j] >> 32)), all.top, s.inv) * up / (double)f.whole));
            }
            n += (uint32_t)__popcll(m);
        }
        if (t == 0) w.out[0] = min(n, SM_FEW);
        return;
    }
    if (listed_kind) {      // the parts' units that stay: above the listed bins, and the list's
        uint64_t *const units = &aheads[0][0];
        static_assert(4 * SM_RANKED >= SM_PARTS, "room for the parts");
        if (t < p.parts) units[t] = __hip_atomic_load(w.kept + t, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
#pragma unroll 1
        for (uint32_t j = t; j < list.n; j += SM_THREADS)
            if (in(j)) atomicAdd((unsigned long long *)units + ~(uint32_t)list.order[j] / (SM_IDS * p.rounds), (unsigned long long)list.unit[j]);
        __syncthreads();
        const uint64_t mine = t < p.parts ? units[t] : 0, before = sm_scan(mine, &total, tmp);
        want = (uint64_t)((double)s.u * (double)total);
        if (want >= before && want < before + mine) { found.kabove = t; found.ksum = before; }
        __syncthreads();
        mine_part = found.kabove;
        want -= found.ksum;
    }
    sm_pick(a, p, r, mine_part, al, s, all.top, up, (double)total, here, want, tmp, &least, [&](float x, uint32_t i) {
        if (!listed_kind) return true;
        const uint32_t y = sm_bin(x, all.top, scale);
        return y < b.first || ((y == b.kbin || (p_on && y <= b.phi)) && ((uint64_t)sm_key(x) << 32 | (uint32_t)~i) >= f.border);
    });
}

// ---- 4
__global__ void __launch_bounds__(SM_THREADS) k_sample_last(sgk_sample_args a, sm_plan p, int al) {
    __shared__ uint64_t tmp[SM_WAVES], sums[3][SM_WAVES];
    __shared__ uint32_t least;
    __shared__ sm_list list;
    const uint32_t t = threadIdx.x, part = blockIdx.x, r = blockIdx.y;
    const sm_row w = sm_at(p, r);
    const sm_set s = sm_settings(a, p, r);
    const sm_all all = *w.all;
    const bool zero = !all.ok || s.few;
    if (!all.ok && part == 0 && t == 0) a.token[r] = SM_NONE;
    const bool k_on = s.top_k && s.top_k < all.ok, p_on = s.top_p < 1.0f;
    if (all.ok && (s.few || k_on || p_on) && *w.listed > SM_LIST) {
        if (part == 0) sm_slow(a, r, s, &list);
        return;
    }
    if (zero) {
        if (!a.probs) return;
        for (uint32_t m = 0; m < p.rounds; m++) {
            const uint64_t i0 = ((uint64_t)part * p.rounds + m) * SM_IDS;
            for (uint32_t e = t; e < SM_IDS && i0 + e < a.vocab; e += SM_THREADS) a.probs[(uint64_t)r * a.vocab + i0 + e] = 0.0f;
        }
        __syncthreads();
        if (all.ok && t < w.out[0]) {
            const uint32_t id = w.out[1 + 2 * t];
            if (id / (SM_IDS * p.rounds) == part) a.probs[(uint64_t)r * a.vocab + id] = __uint_as_float(w.out[2 + 2 * t]);
        }
        return;
    }
    if (!k_on && !p_on) return;
    const double up = sm_unit(all.sum);
    const sm_border b = *w.border;
    const float scale = sm_bin_scale(s, all);
    sm_fetch(list, w, s, all, up, scale);
    const sm_result f = sm_search(list, s, all, b, up, false);
    // the units that stay: above the listed bins by parts, and the list's
    const uint32_t i0 = part * p.rounds * SM_IDS, i1 = i0 + p.rounds * SM_IDS;
    uint64_t whole = 0, before = 0, mine = 0;
    if (t < p.parts) {
        const uint64_t q = w.kept[t];
        whole = q;
        if (t < part) before = q;
        if (t == part) mine = q;
    }
    for (uint32_t j = t; j < list.n; j += SM_THREADS)
        if (list.order[j] >= f.border && !(list.bin[j] & SM_LOW)) {
            const uint32_t id = ~(uint32_t)list.order[j];
            whole += list.unit[j];
            if (id < i0) before += list.unit[j];
            else if (id < i1) mine += list.unit[j];
        }
    whole = wave_sum(whole);
    before = wave_sum(before);
    mine = wave_sum(mine);
    if ((t & 63) == 0) { sums[0][t >> 6] = whole; sums[1][t >> 6] = before; sums[2][t >> 6] = mine; }
    __syncthreads();
    whole = before = mine = 0;
#pragma unroll
    for (int i = 0; i < SM_WAVES; i++) { whole += sums[0][i]; before += sums[1][i]; mine += sums[2][i]; }
    const uint64_t want = (uint64_t)((double)s.u * (double)whole), border = f.border;
    sm_pick(a, p, r, part, al, s, all.top, up, (double)whole, want >= before && want < before + mine, want - before, tmp, &least,
            [&](float x, uint32_t i) {
                const uint32_t y = sm_bin(x, all.top, scale);
                return y < b.first || ((y == b.kbin || (p_on && y <= b.phi)) && ((uint64_t)sm_key(x) << 32 | (uint32_t)~i) >= border);
            });
}

// Parts of a row: one round each until the rows have SM_WGS of them together.
static sm_plan sm_plan_of(uint32_t vocab, uint32_t rows, void *at) {
    sm_plan p;
    const uint64_t chunks = ((uint64_t)vocab + SM_IDS - 1) / SM_IDS, most = min(SM_PARTS, max(SM_WGS / rows, 8u));
    p.rounds = (uint32_t)((chunks + most - 1) / most);
    p.parts = (uint32_t)((chunks + p.rounds - 1) / p.rounds);
    p.row_bytes = sm_row_bytes(p.parts);
    p.at = (char *)at;
    return p;
}
// Rows go by SM_ROWS at a time, so that the scratch memory has an end.
#define SM_ROWS 1024u
extern "C" uint64_t sgk_sample_scratch(const sgk_sample_args *a) { return sm_plan_of(a->vocab, min(a->rows, SM_ROWS), NULL).row_bytes * min(a->rows, SM_ROWS); }
extern "C" hipError_t sgk_sample(const sgk_sample_args *a, void *scratch, hipStream_t s, hipEvent_t done) {
    const sm_plan p = sm_plan_of(a->vocab, min(a->rows, SM_ROWS), scratch);
    const int al = !(((uintptr_t)a->x | (uintptr_t)a->probs) & 15) && a->vocab % 4 == 0;
    for (uint32_t r = 0; r < a->rows; r += SM_ROWS) {
        sgk_sample_args b = *a;
        b.x += (uint64_t)r * a->vocab;
        b.settings += 4ull * r;
        b.u += r;
        b.token += r;
        if (b.probs) b.probs += (uint64_t)r * a->vocab;
        b.rows = min(a->rows - r, SM_ROWS);
        const dim3 grid(p.parts, b.rows);
        launch(k_sample_parts, grid, SM_THREADS, s, (hipEvent_t)NULL, b, p, al);
        launch(k_sample_count, grid, SM_THREADS, s, (hipEvent_t)NULL, b, p, al);
        const hipEvent_t ev = r + SM_ROWS < a->rows ? (hipEvent_t)NULL : done;
        if (!b.probs) {
            launch(k_sample_border<true>, grid, SM_THREADS, s, ev, b, p, al);
            continue;
        }
        launch(k_sample_border<false>, grid, SM_THREADS, s, (hipEvent_t)NULL, b, p, al);
        launch(k_sample_last, grid, SM_THREADS, s, ev, b, p, al);
    }
    return hipGetLastError();
}
