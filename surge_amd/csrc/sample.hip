// sample.hip - a token a row from logits under temperature, top-k, top-p and
// min-p, by a given random number. The launcher is declared in kernels.h; its
// host checks are in hip.c.
#include "devutil.h"
#include "kernels.h"

// ---------------------------------------------------------------------------
// An id's weight is exp((x - max) / temperature), in 64 bits. Sums of weights
// are integers in units of the row's whole sum / 2^61 or so: whatever order the
// additions come in, the sums, the kept ids and the token are the same.
// A workgroup per row; the borders of top-k and top-p by the digits of the
// logits' keys, 8 bits a pass over the row.
// ---------------------------------------------------------------------------
#define SM_THREADS 1024
#define SM_NONE 0xFFFFFFFFu

// Rising with x; 0 for what is never chosen (NaN, -inf).
__device__ __forceinline__ uint32_t sm_key(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);       // -0 as 0
    return x > -INFINITY ? (b & 0x80000000u ? ~b : b | 0x80000000u) : 0;
}
__device__ __forceinline__ double sm_weight(float x, float top, double inv) {
    return x == top ? 1.0 : x > -INFINITY ? exp(((double)x - (double)top) * inv) : 0.0;
}
__device__ __forceinline__ uint64_t sm_units(double w, double up) { return w > 0.0 ? max((uint64_t)1, (uint64_t)rint(w * up)) : 0; }
template <typename T>
__device__ __forceinline__ T sm_sum(T v, T *tmp) {
    for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) tmp[threadIdx.x >> 6] = v;
    __syncthreads();
    T r = 0;
    for (int i = 0; i < SM_THREADS / 64; i++) r += tmp[i];
    return r;
}
template <typename T>
__device__ __forceinline__ T sm_scan(T v, T *total, T *tmp) {      // exclusive
    const uint32_t t = threadIdx.x;
    T x = v;
    for (uint32_t d = 1; d < 64; d <<= 1) {
        const T y = __shfl_up(x, d);
        if ((t & 63) >= d) x += y;
    }
    __syncthreads();
    if ((t & 63) == 63) tmp[t >> 6] = x;
    __syncthreads();
    T before = 0, all = 0;
    for (uint32_t i = 0; i < SM_THREADS / 64; i++) {
        if (i < t >> 6) before += tmp[i];
        all += tmp[i];
    }
    *total = all;
    return before + x - v;
}

__global__ void __launch_bounds__(SM_THREADS) k_sample(sgk_sample_args a) {
    __shared__ uint64_t hist[256], tmp[SM_THREADS / 64], pick[2];
    __shared__ uint32_t tmp32[SM_THREADS / 64], token;
    const uint32_t t = threadIdx.x, r = blockIdx.x, v = a.vocab;
    const float *x = a.x + (uint64_t)r * v;
    const uint32_t *set = a.settings + 4ull * r;
    float temp = __uint_as_float(set[0]), top_p = __uint_as_float(set[2]);
    uint32_t top_k = set[1];
    const float min_p = __uint_as_float(set[3]);
    float u = a.u[r];
    u = u > 0.0f ? fminf(u, 0x1.fffffep-1f) : 0.0f;
    if (!(temp > 0.0f)) { temp = 1.0f; top_k = 1; }
    uint32_t best = 0, ok = 0;
    for (uint32_t i = t; i < v; i += SM_THREADS) {
        const uint32_t key = sm_key(x[i]);
        best = max(best, key);
        ok += key != 0;
    }
    for (int d = 1; d < 64; d <<= 1) best = max(best, (uint32_t)__shfl_xor(best, d));
    if ((t & 63) == 0) tmp32[t >> 6] = best;
    __syncthreads();
    for (int i = 0; i < SM_THREADS / 64; i++) best = max(best, tmp32[i]);
    __syncthreads();
    ok = sm_sum(ok, tmp32);
    float *probs = a.probs ? a.probs + (uint64_t)r * v : NULL;
    if (!ok) {
        if (t == 0) a.token[r] = SM_NONE;
        if (probs) for (uint32_t i = t; i < v; i += SM_THREADS) probs[i] = 0.0f;
        return;
    }
    const float top = __uint_as_float(best & 0x80000000u ? best ^ 0x80000000u : ~best);
    const double inv = 1.0 / (double)temp;
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
    double sum = sm_sum(part, (double *)tmp);
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
extern "C" hipError_t sgk_sample(const sgk_sample_args *a, hipStream_t s, hipEvent_t done) {
    launch(k_sample, dim3(a->rows), SM_THREADS, s, done, *a);
    return hipGetLastError();
}
