// Sampling with temperature, top-k, nucleus (top-p) and min-p at given uniforms (gfx950), for vocabularies of up to 2^18 symbols.
//
// A row's entries in the order (logit descending, index ascending) have the weights w_j = exp((x_j - max x) / temperature).  Every one
// of the four rules keeps a prefix of that order, so the kept set is the shortest of them and what is needed are ranks and
// cumulative weights at a few places of the order, not the order itself: nothing is sorted.  Two searches are enough,
//     mass of the first r entries (top-k)      and      first entry whose cumulative weight exceeds T (nucleus, draw),
// and both walk one histogram of 2048 bins over (max x - x) / temperature and then look into the single bin that holds the border.
//
// Weights are whole multiples of 2^-45 in 64 bits (computed in f64): their sums do not depend on the order in which LDS
// atomics arrive, so a call repeats bit for bit, and 2^18 of them cannot overflow.  A pick next to a border between two entries
// needs about that many bits: the cumulative weights of a flat row lie 2^-18 apart, and f32 sums would move one pick in a few thousand.
#include "me_common.h"
#include <math.h>

namespace {

typedef unsigned long long u64;

constexpr int NB = 2048;                    // bins of a search level
constexpr int NL = 1024;                    // entries of a bin that are compared with each other directly
constexpr int FRAC = 45;                    // weight unit 2^-45

struct SampleArgs {
    const float* logits; int ld, V;
    const int32_t* special; int n_special;
    const float* temp;
    int top_k; float top_p;
    double y_min;                           // log2(min_p)
    const float* u;
    int64_t* out; int32_t* choices;
    // a step of a device-resident loop (prev != NULL): temperature from the token just fed, uniform from a table, repeat counter
    const int64_t* prev; const uint8_t* is_timeshift; float* repeats; const int32_t* pos;
    int pos0, u_ld; float temp_note, temp_rest, penalty;
};

// order-preserving image of (x, j): greater = earlier in the order
ME_DEV u64 word_of(float x, int j) {
    uint32_t b = __float_as_uint(x + 0.f);                    // + 0: one zero
    b ^= (b >> 31) ? 0xffffffffu : 0x80000000u;
    return ((u64)b << 32) | (0xffffffffu - (uint32_t)j);
}

// 2^y (y <= 0) in units of 2^-45, rounded to nearest: 2^f on [-1/2, 1/2] by its Taylor series (13 terms: below 2^-50), the
// scaling exact, and the conversion by adding 2^52 (the integer is then the mantissa)
ME_DEV u64 weight_of(double y) {
    if (!(y > -(double)(FRAC + 2))) return 0;
    const double n = rint(y), r = (y - n) * 0.693147180559945309417;
    double p = 1.0 / 479001600.0;
    p = fma(p, r, 1.0 / 39916800.0); p = fma(p, r, 1.0 / 3628800.0); p = fma(p, r, 1.0 / 362880.0); p = fma(p, r, 1.0 / 40320.0);
    p = fma(p, r, 1.0 / 5040.0);     p = fma(p, r, 1.0 / 720.0);     p = fma(p, r, 1.0 / 120.0);    p = fma(p, r, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);        p = fma(p, r, 0.5);             p = fma(p, r, 1.0);            p = fma(p, r, 1.0);
    const double scale = __longlong_as_double((long long)((int)n + FRAC + 1023) << 52);
    return (u64)(__double_as_longlong(fma(p, scale, 0x1p52)) - __double_as_longlong(0x1p52));
}

template <int NT> struct Shared {
    uint32_t cnt[NB];                       // level 0: per bin, then entries before it
    u64 mass[NB];
    uint32_t cnt1[NB];                      // deeper levels
    union {
        u64 mass1[NB];
        struct { u64 lw[NL], lm[NL]; };     // the last bin's entries (word, weight): the level above has been read by then
    };
    u64 r64[NT / 64], found_mass, found_word;
    uint32_t r32[NT / 64], found_bin, found_rank, n_list;
};

template <int NT> ME_DEV u64 block_sum64(Shared<NT>& s, u64 v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s.r64[threadIdx.x >> 6] = v;
    __syncthreads();
    u64 t = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) t += s.r64[w];
    return t;
}
template <int NT> ME_DEV u64 block_max64(Shared<NT>& s, u64 v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) { const u64 x = __shfl_xor(v, o); v = x > v ? x : v; }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s.r64[threadIdx.x >> 6] = v;
    __syncthreads();
    u64 t = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) t = s.r64[w] > t ? s.r64[w] : t;
    return t;
}

// per-bin counts and masses -> what lies before each bin; returns the totals
template <int NT> ME_DEV void scan_bins(Shared<NT>& s, uint32_t* cnt, u64* mass, uint32_t& n_all, u64& m_all) {
    constexpr int PB = NB / NT;
    const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
    uint32_t c[PB], cs = 0;
    u64 m[PB], ms = 0;
#pragma unroll
    for (int i = 0; i < PB; ++i) { c[i] = cnt[tid * PB + i]; m[i] = mass[tid * PB + i]; cs += c[i]; ms += m[i]; }
    uint32_t ci = cs;
    u64 mi = ms;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t x = __shfl_up(ci, o);
        const u64 y = __shfl_up(mi, o);
        if (lane >= o) { ci += x; mi += y; }
    }
    __syncthreads();
    if (lane == 63) { s.r32[wid] = ci; s.r64[wid] = mi; }
    __syncthreads();
    n_all = 0; m_all = 0;
    uint32_t cb = 0;
    u64 mb = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) {
        if (w == wid) { cb = n_all; mb = m_all; }
        n_all += s.r32[w];
        m_all += s.r64[w];
    }
    cb += ci - cs;
    mb += mi - ms;
#pragma unroll
    for (int i = 0; i < PB; ++i) {
        cnt[tid * PB + i] = cb; mass[tid * PB + i] = mb;
        cb += c[i]; mb += m[i];
    }
    __syncthreads();
}

// NT threads per row.  ROW: the row stays in LDS after the first pass (V <= ROW_MAX); else every pass reads it again (from L2)
constexpr int ROW_MAX = 26624;
template <int NT, bool ROW>
__global__ __launch_bounds__(NT) void sample_minp_kernel(const SampleArgs a) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    Shared<NT>& s = *reinterpret_cast<Shared<NT>*>(smem);
    uint32_t* barred = reinterpret_cast<uint32_t*>(smem + sizeof(Shared<NT>));        // !ROW: one bit per symbol
    float* row = reinterpret_cast<float*>(smem + sizeof(Shared<NT>));                 // ROW: the logits
    const int tid = threadIdx.x, b = blockIdx.x, V = a.V;
    const float* lg = a.logits + (size_t)b * a.ld;
    constexpr int U = ROW ? 4 : 8;                            // entries of a thread in flight

    // every entry once: NaN -> 0, special ids -> -inf
    auto each = [&](auto&& f) {
        for (int j0 = tid; j0 < V; j0 += NT * U) {
            float x[U];
#pragma unroll
            for (int q = 0; q < U; ++q) { const int j = min(j0 + q * NT, V - 1); x[q] = ROW ? row[j] : lg[j]; }
#pragma unroll
            for (int q = 0; q < U; ++q) {
                const int j = j0 + q * NT;
                if (j < V) {
                    float v = x[q];
                    if (!ROW) { if (v != v) v = 0.f; if ((barred[j >> 5] >> (j & 31)) & 1u) v = -INFINITY; }
                    f(v, j);
                }
                __builtin_amdgcn_sched_barrier(0);            // the entries' f64 chains stay apart (the waves hide them): few registers
            }
        }
    };
    if constexpr (ROW) {
        constexpr int L = 8;
        for (int j0 = tid; j0 < V; j0 += NT * L) {
            float x[L];
#pragma unroll
            for (int q = 0; q < L; ++q) x[q] = lg[min(j0 + q * NT, V - 1)];
#pragma unroll
            for (int q = 0; q < L; ++q) if (j0 + q * NT < V) row[j0 + q * NT] = x[q] != x[q] ? 0.f : x[q];
        }
        __syncthreads();
        for (int i = tid; i < a.n_special; i += NT) { const int j = a.special[i]; if (j >= 0 && j < V) row[j] = -INFINITY; }
    } else {
        for (int i = tid; i < (V + 31) / 32; i += NT) barred[i] = 0;
        __syncthreads();
        for (int i = tid; i < a.n_special; i += NT) { const int j = a.special[i]; if (j >= 0 && j < V) atomicOr(&barred[j >> 5], 1u << (j & 31)); }
    }
    __syncthreads();

    // ---- temperature and uniform of the row (step form: the f32 operations of generate.py's sampling_temperature(), unfused)
    float temp, u;
    if (a.prev) {
        const int64_t pt = a.prev[b];
        temp = pt >= 0 && pt < V && a.is_timeshift[pt] ? a.temp_note : a.temp_rest;
        if (a.penalty > 0.f) {
            const float mult = fmaxf(__fmul_rn(logf(__fdiv_rn(__fadd_rn(a.repeats[b], 1.f), 4.f)), a.penalty), 0.f);
            temp = __fadd_rn(temp, __fmul_rn(mult, temp));
        }
        u = a.u[(size_t)(a.pos[0] - a.pos0) * a.u_ld + b];
    } else {
        temp = a.temp[b];
        u = a.u[b];
    }

    float mx = -INFINITY;
    each([&](float v, int) { mx = fmaxf(mx, v); });
    mx = wave_max(mx);
    if ((tid & 63) == 0) s.r32[tid >> 6] = __float_as_uint(mx);
    for (int i = tid; i < NB; i += NT) { s.cnt[i] = 0; s.mass[i] = 0; }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) mx = fmaxf(mx, __uint_as_float(s.r32[w]));

    auto finish = [&](int64_t id, int n) {                    // one thread
        a.out[b] = id;
        if (a.choices) a.choices[b] = n;
        if (a.prev) { const float rc = a.repeats[b]; a.repeats[b] = n <= 2 ? rc + 1.f : floorf(rc * 0.5f); }      // generate.py:186-189
    };
    if (mx == -INFINITY) {                                    // nothing to choose from
        if (tid == 0) finish(0, 0);
        return;
    }
    // exponents: y = (x - max) / temperature * log2 e in f64; equal values (two infinities too) give 0
    const double c2 = 1.4426950408889634074 / (double)temp;
    const float bin_c = (float)NB / 32.f / temp;
    auto exponent = [&](float v) -> double { return v == mx ? 0.0 : ((double)v - (double)mx) * c2; };
    auto bin_of = [&](float v) -> int { return v == mx ? 0 : (int)fminf((mx - v) * bin_c, (float)(NB - 1)); };

    // ---- histogram; what min-p and a positive weight leave is a threshold on y: counted on the way
    const double y_min = a.y_min;
    uint32_t n_keep = 0;
    u64 m_keep = 0;
    each([&](float v, int) {
        const double y = exponent(v);
        const u64 w = weight_of(y);
        const bool keep = y >= y_min && y > -1075.0;          // exp() of 64 bits is 0 from 2^-1075 on
        n_keep += keep;
        m_keep += keep ? w : 0;
        const int bin = bin_of(v);
        atomicAdd(&s.cnt[bin], 1u);
        if (w) atomicAdd(&s.mass[bin], w);
    });
    n_keep = (uint32_t)block_sum64(s, (u64)n_keep);
    m_keep = block_sum64(s, m_keep);
    uint32_t n_all;
    u64 m_all;
    scan_bins<NT>(s, s.cnt, s.mass, n_all, m_all);

    // ---- search: by_rank: the mass of the first `rank` entries; else the first entry whose cumulative weight exceeds `limit`
    //      (its word, its rank, the mass before it)
    auto search = [&](bool by_rank, uint32_t rank, u64 limit, u64& word, uint32_t& at, u64& before) {
        uint32_t* cnt = s.cnt;
        u64* mass = s.mass;
        uint32_t total = n_all, c0 = 0;                       // entries and mass before the window of this level
        u64 mtotal = m_all, m0 = 0;
        u64 hi = 0, lo = 0;
        int shift = 0, level = 0, bin0 = 0;
        while (true) {
            for (int i = tid; i < NB; i += NT) {
                const uint32_t cb = c0 + cnt[i], ce = c0 + (i + 1 < NB ? cnt[i + 1] : total);
                const u64 mb = m0 + mass[i], me = m0 + (i + 1 < NB ? mass[i + 1] : mtotal);
                if (by_rank ? (cb < rank && rank <= ce) : (mb <= limit && limit < me)) s.found_bin = (uint32_t)i;
            }
            __syncthreads();
            const int bin = (int)s.found_bin;
            const uint32_t cb = c0 + cnt[bin], n = c0 + (bin + 1 < NB ? cnt[bin + 1] : total) - cb;
            const u64 mb = m0 + mass[bin];
            if (level == 0) bin0 = bin;
            else { const u64 top = hi - ((u64)bin << shift); lo = max(lo, top - (((u64)1 << shift) - 1)); hi = top; }
            c0 = cb;
            m0 = mb;
            __syncthreads();                                  // found_bin, cnt, mass have been read
            auto inside = [&](float v, u64 w) { return level == 0 ? bin_of(v) == bin0 : w <= hi && w >= lo; };
            if (n <= NL) {
                if (tid == 0) s.n_list = 0;
                __syncthreads();
                each([&](float v, int j) {
                    const u64 w = word_of(v, j);
                    if (inside(v, w)) s.lw[atomicAdd(&s.n_list, 1u)] = w;
                });
                __syncthreads();
                for (uint32_t e = tid; e < n; e += NT) {
                    uint32_t bits = (uint32_t)(s.lw[e] >> 32);
                    bits ^= (bits >> 31) ? 0x80000000u : 0xffffffffu;
                    s.lm[e] = weight_of(exponent(__uint_as_float(bits)));
                }
                __syncthreads();
                for (uint32_t e = tid; e < n; e += NT) {
                    const u64 me = s.lw[e], own = s.lm[e];
                    uint32_t r = 0;
                    u64 cum = own;
#pragma clang loop unroll_count(4)
                    for (uint32_t k = 0; k < n; ++k) { const bool ahead = s.lw[k] > me; r += ahead; cum += ahead ? s.lm[k] : 0; }
                    const bool hit = by_rank ? c0 + r + 1 == rank : (m0 + cum > limit && m0 + cum - own <= limit);
                    if (hit) { s.found_word = me; s.found_rank = c0 + r; s.found_mass = by_rank ? m0 + cum : m0 + cum - own; }
                }
                __syncthreads();
                word = s.found_word;
                at = s.found_rank;
                before = s.found_mass;
                __syncthreads();
                return;
            }
            // too many for that: the entries between the bin's first and last word, cut into 2048 pieces of the word's range (words
            // differ, so a few levels end at one entry each)
            u64 wmax = 0, wmin = 0;                           // wmin as the maximum of the complement
            each([&](float v, int j) { const u64 w = word_of(v, j); if (inside(v, w)) { wmax = max(wmax, w); wmin = max(wmin, ~w); } });
            hi = block_max64(s, wmax);
            lo = ~block_max64(s, wmin);
            level = 1;
            shift = 0;
            while (((hi - lo) >> shift) >= NB) ++shift;
            for (int i = tid; i < NB; i += NT) { s.cnt1[i] = 0; s.mass1[i] = 0; }
            __syncthreads();
            each([&](float v, int j) {
                const u64 w = word_of(v, j);
                if (w <= hi && w >= lo) {
                    const int i = (int)((hi - w) >> shift);
                    const u64 m = weight_of(exponent(v));
                    atomicAdd(&s.cnt1[i], 1u);
                    if (m) atomicAdd(&s.mass1[i], m);
                }
            });
            __syncthreads();
            cnt = s.cnt1;
            mass = s.mass1;
            scan_bins<NT>(s, cnt, mass, total, mtotal);
        }
    };

    // ---- top-k, then min-p, then the nucleus, then the draw
    u64 word = 0, mass = 0, tot = m_all, tot_k = m_all, limit = 0;
    uint32_t at = 0, n = n_all;
#pragma clang loop unroll(disable)
    for (int phase = 0; phase < 3; ++phase) {
        if (phase == 0) {
            if (a.top_k <= 0 || (uint32_t)a.top_k >= n) continue;
            n = (uint32_t)a.top_k;
        } else if (phase == 1) {
            tot_k = tot;
            if (n_keep < n) { n = n_keep; tot = m_keep; }
            limit = (u64)((double)a.top_p * (double)tot_k);
            if (!(a.top_p > 0.f && a.top_p < 1.f) || limit >= tot) continue;      // the nucleus holds all that the others keep
        } else {
            const double ut = u > 0.f ? (double)u * (double)tot : 0.0;
            limit = ut < (double)tot ? min((u64)ut, tot - 1) : tot - 1;           // u >= 1: the last entry that has a weight
        }
        search(phase == 0, n, limit, word, at, mass);
        if (phase == 0) tot = mass;
        if (phase == 1) { n = at > 0 ? at : 1; tot = at > 0 ? mass : (u64)1 << FRAC; }        // its first entry always stays
    }
    if (tid == 0) finish((int64_t)(0xffffffffu - (uint32_t)word), (int)n);
}

template <int NT, bool ROW> int launch(const SampleArgs& a, int B, hipStream_t st) {
    const size_t lds = sizeof(Shared<NT>) + (ROW ? (size_t)a.V * 4 : (size_t)(a.V + 31) / 32 * 4);
    static bool raised[64] = {};                              // per device: more than 64 KB of LDS has been allowed
    int dev = 0;
    (void)hipGetDevice(&dev);
    if (lds > 65536 && !(dev >= 0 && dev < 64 && raised[dev])) {
        if (hipFuncSetAttribute(reinterpret_cast<const void*>(&sample_minp_kernel<NT, ROW>), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024) != hipSuccess)
            return ME_ERR_LAUNCH;
        if (dev >= 0 && dev < 64) raised[dev] = true;
    }
    sample_minp_kernel<NT, ROW><<<B, NT, lds, st>>>(a);
    return me_launch_status();
}

int sample_call(const SampleArgs& a, int B, hipStream_t st) {
    if (a.V <= 4096) return launch<256, true>(a, B, st);
    if (a.V <= ROW_MAX) return launch<1024, true>(a, B, st);
    return launch<1024, false>(a, B, st);
}

}  // namespace

extern "C" {

int me_sample_minp(const float* logits, int ld, int V, const int32_t* special, int n_special, const float* temp, int top_k, float top_p,
                   float min_p, const float* u, int64_t* out_ids, int32_t* n_choices, int B, void* stream) {
    me_clear_error();
    if (!logits || !temp || !u || !out_ids || (n_special > 0 && !special)) return ME_ERR_NULL;
    if (B < 0 || V <= 0 || V > ME_SAMPLE_MAX_VOCAB || ld < V || n_special < 0 || !(min_p >= 0.f && min_p <= 1.f)) return ME_ERR_BAD_SHAPE;
    if (B == 0) return ME_OK;
    SampleArgs a = {logits, ld, V, special, n_special, temp, top_k, top_p, log2((double)min_p), u, out_ids, n_choices, nullptr, nullptr, nullptr, nullptr, 0, 0, 0.f, 0.f, 0.f};
    return sample_call(a, B, (hipStream_t)stream);
}

int me_sample_minp_step(const float* logits, int ld, int V, const int32_t* special, int n_special, const int64_t* prev_tok,
                        const uint8_t* is_timeshift, float* repeat_counts, float temp_note, float temp_rest, float penalty_coeff, int top_k,
                        float top_p, float min_p, const float* u_table, int u_ld, const int32_t* pos, int pos0, int64_t* out_ids,
                        int32_t* n_choices, int B, void* stream) {
    me_clear_error();
    if (!logits || !prev_tok || !is_timeshift || !repeat_counts || !u_table || !pos || !out_ids || (n_special > 0 && !special)) return ME_ERR_NULL;
    if (B < 0 || V <= 0 || V > ME_SAMPLE_MAX_VOCAB || ld < V || u_ld < B || n_special < 0 || !(min_p >= 0.f && min_p <= 1.f)) return ME_ERR_BAD_SHAPE;
    if (B == 0) return ME_OK;
    SampleArgs a = {logits, ld, V, special, n_special, nullptr, top_k, top_p, log2((double)min_p), u_table, out_ids, n_choices, prev_tok, is_timeshift, repeat_counts,
                    pos, pos0, u_ld, temp_note, temp_rest, penalty_coeff};
    return sample_call(a, B, (hipStream_t)stream);
}

}  // extern "C"
