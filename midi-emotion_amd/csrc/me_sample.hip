// Sampling with temperature, top-k, nucleus (top-p) and min-p at given uniforms (gfx950), for vocabularies of up to 2^18 symbols.
//
// A row's entries in the order (logit descending, index ascending) have the weights w_j = exp((x_j - max x) / temperature).  Every one
// of the four rules keeps a prefix of that order, so the kept set is the shortest of them and what is needed are ranks and
// cumulative weights at a few places of the order, not the order itself: nothing is sorted.  Two searches are enough,
//     mass of the first r entries (top-k)      and      first entry whose cumulative weight exceeds T (nucleus, draw),
// and both walk one histogram of 1024 bins over (max x - x) / temperature and then look into the single bin that holds the border.
//
// Weights are whole multiples of 2^-45 in 64 bits (computed in f64): their sums do not depend on the order in which LDS
// atomics arrive, so a call repeats bit for bit, and 2^18 of them cannot overflow.  A pick next to a border between two entries
// needs about that many bits: the cumulative weights of a flat row lie 2^-18 apart, and f32 sums would move one pick in a few thousand.
//
// What bounds it: not the bytes (4 V a row) but instructions and barriers: the f64 weight of every entry, about 30 instructions, on
// however many CUs share a row, and the chain of block-wide steps of the two or three searches.  Rows of up to 32512 symbols take one block, the
// row, bins and lists in its LDS.  Wider ones take four launches: the chunks' maxima; the chunks' histograms; the members of
// the bins that can hold one of the borders (known up to a bin or two from the histogram alone), gathered by all chunks; and one block per
// row that finishes on those few entries.  Measured, us a call in a graph, top_p 0.9 and min_p 0.05 / top_k 200, top_p 0.95 and min_p 0.02:
//   one block, 256 threads:   4 x 1018: 7.7 / 11.1,  64 x 2048: 10.5 / 14.4,  512 x 1018: 10.5 / 14.4
//   one block, 1024 threads:  64 x 32000: 23.6 / 24.2 (0.35 TB/s: 64 of 256 CUs),  256 x 32512: 27.8 / 28.1 (1.2 TB/s)
//   four launches:            1 x 131071: 27.8 / 32.4,  128 x 131071: 64.8 / 77.0 (1.0 TB/s; the row is read three times, from the
//                             last-level cache: maxima 12, histograms 29, gathering 21, finish 15 us)
// Rows whose logits lie close together put more than 4096 entries into a border's bin; the last launch then walks the row itself, one block for
// each, twice for every level of a search: 128 x 131071 of equal logits 1065 / 1524 us, of deviation 0.1 (temperature 1) 1173 / 93; 64 x 32000: 213 / 288, 113 / 41.
#include "me_common.h"
#include <algorithm>
#include <math.h>

namespace {

typedef unsigned long long u64;

constexpr int NB = 1024;                    // bins of a search level; level 0: 32 per unit of (max - x) / temperature
constexpr int NB1 = 256;                    // pieces of a bin that holds many
constexpr int CL = 512;                     // entries of a bin that are collected in one walk over the row
constexpr int SL = 1024;                    // entries up to top-k's border that take the row's place
constexpr int NL = 128;                     // entries that are compared with each other directly
constexpr int GL = 4096;                    // gathered entries of a wide row
constexpr int FRAC = 45;                    // weight unit 2^-45
// 32512: the row, the bins and the lists fill 160 KB of LDS.  Up to there one block is faster at every batch measured, although
// few rows leave CUs idle: 32512 symbols in one block / 32513 in four launches, us: 1 row 22.4 / 25.5, 8: 23.0 / 28.3, 64: 25.0 / 38.4, 512: 52.9 / 67.2
// (top_p 0.9, min_p 0.05; nearest to each other for a single row with top_p 0.98, min_p 0.001: 25.6 / 26.2)
constexpr int ONE_BLOCK = ME_SAMPLE_ONE_BLOCK;
constexpr int MAX_SPLIT = 16;               // chunks of a wide row at most: every later block reads all chunks' histograms

struct SampleArgs {
    const float* logits; int ld, V;
    const int32_t* special; int n_special;
    const float* temp;
    int top_k; float top_p;
    double y_min;                           // least_exponent(min_p)
    const float* u;
    int64_t* out; int32_t* choices;
    // a step of a device-resident loop (prev != NULL): temperature from the token just fed, uniform from a table, repeat counter
    const int64_t* prev; const uint8_t* is_timeshift; float* repeats; const int32_t* pos;
    int pos0, u_ld; float temp_note, temp_rest, penalty;
    // wide rows: the workspace, the chunks
    char* ws; int splits, chunk;
};

// workspace of a wide row (16-byte multiples); written before it is read by every call
struct RowWs {
    u64* mass;                              // [splits][NB]
    uint32_t* cnt;                          // [splits][NB]
    u64* m_keep;                            // [MAX_SPLIT]
    u64* m_tot;                             // [MAX_SPLIT]
    uint32_t* n_keep;                       // [MAX_SPLIT]
    float* mx;                              // [MAX_SPLIT]
    uint32_t* n_list;                       // [4]
    int* ranges;                            // [8]: the gathered bins
    u64* list;                              // [GL]
};
__host__ __device__ inline size_t row_ws_bytes(int splits) { return (size_t)splits * NB * 12 + MAX_SPLIT * 24 + 16 + 32 + GL * 8; }
ME_DEV RowWs row_ws(const SampleArgs& a, int b) {
    char* p = a.ws + (size_t)b * row_ws_bytes(a.splits);
    RowWs w;
    w.mass = reinterpret_cast<u64*>(p); p += (size_t)a.splits * NB * 8;
    w.cnt = reinterpret_cast<uint32_t*>(p); p += (size_t)a.splits * NB * 4;
    w.m_keep = reinterpret_cast<u64*>(p); p += MAX_SPLIT * 8;
    w.m_tot = reinterpret_cast<u64*>(p); p += MAX_SPLIT * 8;
    w.n_keep = reinterpret_cast<uint32_t*>(p); p += MAX_SPLIT * 4;
    w.mx = reinterpret_cast<float*>(p); p += MAX_SPLIT * 4;
    w.n_list = reinterpret_cast<uint32_t*>(p); p += 16;
    w.ranges = reinterpret_cast<int*>(p); p += 32;
    w.list = reinterpret_cast<u64*>(p);
    return w;
}

// order-preserving image of (x, j): greater = earlier in the order
ME_DEV u64 word_of(float x, int j) {
    uint32_t b = __float_as_uint(x + 0.f);                    // + 0: one zero
    b ^= (b >> 31) ? 0xffffffffu : 0x80000000u;
    return ((u64)b << 32) | (0xffffffffu - (uint32_t)j);
}
ME_DEV float value_of(u64 word) {
    uint32_t b = (uint32_t)(word >> 32);
    b ^= (b >> 31) ? 0x80000000u : 0xffffffffu;
    return __uint_as_float(b);
}
ME_DEV int index_of(u64 word) { return (int)(0xffffffffu - (uint32_t)word); }

// a row's scale: exponents y = (x - max) / temperature * log2 e, weights 2^y, bins.  Straight code: it runs once per entry.
struct Scale {
    float mx, bin_c;
    double mxd, c;                          // 32 log2 e / temperature
    bool inf;                               // an infinite maximum: it alone has a weight (uniform)
    const double* tab;                      // 2^(i / 32)
    ME_DEV void set(float m, float temp, const double* t) {
        mx = m;
        mxd = m;
        inf = m == INFINITY;
        // a temperature that is not positive counts as 0 (the largest entries alone have a weight), an infinite one as the largest number:
        // exponents and bins stay ordered whatever the device memory holds, and 0 times a factor is 0
        const float tp = temp > 0.f ? fminf(temp, 3.402823466e38f) : 0.f;
        bin_c = fminf((float)NB / 32.f / tp, 3.402823466e38f);
        c = fmin(32 * 1.4426950408889634074 / (double)tp, 1e300);
        tab = t;
    }
    ME_DEV double exponent(float v) const { return inf ? (v == mx ? 0.0 : -INFINITY) : ((double)v - mxd) * c; }        // 32 y
    ME_DEV int bin(float v) const { return inf ? (v == mx ? 0 : NB - 1) : (int)fminf((mx - v) * bin_c, (float)(NB - 1)); }
    // an interval of values that holds bins lo .. hi, a little wider: bins fall with the value, and two comparisons cost a fifth of a bin
    ME_DEV void interval(int lo, int hi, float& v_lo, float& v_hi) const {
        const bool any = lo <= hi;
        const float slack = 1e-5f * fabsf(mx), to = (float)(hi + 1) / bin_c;
        const float at = fminf((float)lo / bin_c, 3.402823466e38f);       // differences past 32 bits are in the last bin: it begins no later than there
        v_hi = !any ? -INFINITY : lo == 0 ? INFINITY : inf ? 3.402823466e38f : mx - at * 0.9999f + slack;
        v_lo = !any || (inf && hi < NB - 1) ? INFINITY : hi >= NB - 1 ? -INFINITY : mx - to * 1.0001f - slack;
    }
    // 2^(e / 32) (e <= 0) in units of 2^-45, rounded to nearest: table times the Taylor series of 2^f, |f| <= 1/64 (6 terms: below
    // 2^-48), scaled exactly, converted by adding 2^52 (the integer is then the mantissa); from 2^-47 on, and for what is no number, 0
    ME_DEV u64 weight(double e) const {
        e = fmax(e, -32.0 * (FRAC + 2));
        const double k = rint(e), r = (e - k) * (0.693147180559945309417 / 32);
        const int n = (int)k;
        double p = fma(r, 1.0 / 120.0, 1.0 / 24.0);
        p = fma(p, r, 1.0 / 6.0); p = fma(p, r, 0.5); p = fma(p, r, 1.0); p = fma(p, r, 1.0);
        const double scale = __longlong_as_double((long long)((n >> 5) + FRAC + 1023) << 52);
        return (u64)(__double_as_longlong(fma(p * tab[n & 31], scale, 0x1p52)) - __double_as_longlong(0x1p52));
    }
};
// the exponent from which min-p and a positive weight keep an entry: exp() of 64 bits is 0 from 2^-1075 on
ME_DEV double keep_floor(const SampleArgs& a) {
    return fmax(32 * a.y_min, __longlong_as_double(__double_as_longlong(-1075.0 * 32) - 1));      // the first double above -1075 * 32
}

// temperature and uniform of a row (step form: the f32 operations of generate.py's sampling_temperature(), unfused)
ME_DEV float row_temp(const SampleArgs& a, int b) {
    if (!a.prev) return a.temp[b];
    const int64_t pt = a.prev[b];
    float temp = pt >= 0 && pt < a.V && a.is_timeshift[pt] ? a.temp_note : a.temp_rest;
    if (a.penalty > 0.f) {
        const float mult = fmaxf(__fmul_rn(logf(__fdiv_rn(__fadd_rn(a.repeats[b], 1.f), 4.f)), a.penalty), 0.f);
        temp = __fadd_rn(temp, __fmul_rn(mult, temp));
    }
    return temp;
}
ME_DEV float row_u(const SampleArgs& a, int b) { return a.prev ? a.u[(size_t)(a.pos[0] - a.pos0) * a.u_ld + b] : a.u[b]; }
ME_DEV void finish(const SampleArgs& a, int b, int64_t id, int n) {       // one thread
    a.out[b] = id;
    if (a.choices) a.choices[b] = n;
    if (a.prev) { const float rc = a.repeats[b]; a.repeats[b] = n <= 2 ? rc + 1.f : floorf(rc * 0.5f); }      // generate.py:186-189
}

// top-k cuts; min-p and the nucleus are in force
ME_DEV bool cuts(const SampleArgs& a) { return a.top_k > 0 && a.top_k < a.V; }
ME_DEV bool has_nucleus(const SampleArgs& a) { return a.top_p > 0.f && a.top_p < 1.f; }
// the exponent from which entries are in the histogram: all of them with top-k, else what min-p keeps
ME_DEV double floor_of(const SampleArgs& a) { return cuts(a) ? -INFINITY : keep_floor(a); }

template <int NT> struct __attribute__((aligned(16))) Shared {
    double tab[32];
    uint32_t cnt[NB];                       // level 0: per bin, then entries before it
    u64 mass[NB];
    uint32_t cnt1[NB1];                     // deeper levels
    u64 mass1[NB1];
    u64 lw[CL];                             // a bin's entries
    u64 lm[NL], lc[NL];                     // the last ones: weight, cumulative weight,
    uint32_t lr[NL];                        // rank
    u64 r64[NT / 64], q64[NT / 64], found_mass, found_word;
    uint32_t r32[NT / 64], found_bin, found_rank, n_list;
};

// inclusive sums over a wave's lanes by lane moves of the vector unit (six steps; through LDS each step is a round trip)
template <int CTRL, int ROWS> ME_DEV uint32_t moved(uint32_t x) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xF, false); }
template <int CTRL, int ROWS> ME_DEV u64 moved(u64 x) { return ((u64)moved<CTRL, ROWS>((uint32_t)(x >> 32)) << 32) | moved<CTRL, ROWS>((uint32_t)x); }
template <typename T> ME_DEV T wave_scan(T x) {
    x += moved<0x111, 0xF>(x);                                // 1, 2, 4, 8 lanes on inside the rows of 16
    x += moved<0x112, 0xF>(x);
    x += moved<0x114, 0xF>(x);
    x += moved<0x118, 0xF>(x);
    x += moved<0x142, 0xA>(x);                                // a row's last lane to the next row (rows 1 and 3)
    x += moved<0x143, 0xC>(x);                                // lane 31 to rows 2 and 3
    return x;
}
// three sums at once
template <int NT> ME_DEV void block_sum3(Shared<NT>& s, uint32_t& n, u64& x, u64& y) {
    n = wave_scan(n);
    x = wave_scan(x);
    y = wave_scan(y);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) { s.r32[threadIdx.x >> 6] = n; s.r64[threadIdx.x >> 6] = x; s.q64[threadIdx.x >> 6] = y; }
    __syncthreads();
    n = 0; x = 0; y = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) { n += s.r32[w]; x += s.r64[w]; y += s.q64[w]; }
}
ME_DEV u64 larger(u64 a, u64 b) { return a > b ? a : b; }
ME_DEV u64 wave_top(u64 x) {                                  // in lane 63
    x = larger(x, moved<0x111, 0xF>(x));
    x = larger(x, moved<0x112, 0xF>(x));
    x = larger(x, moved<0x114, 0xF>(x));
    x = larger(x, moved<0x118, 0xF>(x));
    x = larger(x, moved<0x142, 0xA>(x));
    return larger(x, moved<0x143, 0xC>(x));
}
// two maxima at once
template <int NT> ME_DEV void block_max64(Shared<NT>& s, u64& x, u64& y) {
    x = wave_top(x);
    y = wave_top(y);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) { s.r64[threadIdx.x >> 6] = x; s.q64[threadIdx.x >> 6] = y; }
    __syncthreads();
    x = 0; y = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) { x = larger(s.r64[w], x); y = larger(s.q64[w], y); }
}
template <int NT> ME_DEV float block_max(Shared<NT>& s, float v) {
    v = wave_max(v);
    if ((threadIdx.x & 63) == 0) s.r32[threadIdx.x >> 6] = __float_as_uint(v);
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) v = fmaxf(v, __uint_as_float(s.r32[w]));
    return v;
}

// per-bin counts and masses -> what lies before each bin; returns the totals
template <int NT, int N> ME_DEV void scan_bins(Shared<NT>& s, uint32_t* cnt, u64* mass, uint32_t& n_all, u64& m_all) {
    constexpr int PB = N > NT ? N / NT : 1;
    const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
    const bool on = tid * PB < N;
    uint32_t c[PB], cs = 0;
    u64 m[PB], ms = 0;
#pragma unroll
    for (int i = 0; i < PB; ++i) { c[i] = on ? cnt[tid * PB + i] : 0; m[i] = on ? mass[tid * PB + i] : 0; cs += c[i]; ms += m[i]; }
    const uint32_t ci = wave_scan(cs);
    const u64 mi = wave_scan(ms);
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
        if (on) { cnt[tid * PB + i] = cb; mass[tid * PB + i] = mb; }
        cb += c[i]; mb += m[i];
    }
    __syncthreads();
}

// masses alone
template <int NT> ME_DEV void scan_mass(Shared<NT>& s, u64* mass, u64& m_all) {
    constexpr int PB = NB / NT;
    const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
    u64 m[PB], ms = 0;
#pragma unroll
    for (int i = 0; i < PB; ++i) { m[i] = mass[tid * PB + i]; ms += m[i]; }
    const u64 mi = wave_scan(ms);
    __syncthreads();
    if (lane == 63) s.r64[wid] = mi;
    __syncthreads();
    u64 mb = mi - ms;
    m_all = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) { if (w < wid) mb += s.r64[w]; m_all += s.r64[w]; }
#pragma unroll
    for (int i = 0; i < PB; ++i) { mass[tid * PB + i] = mb; mb += m[i]; }
    __syncthreads();
}

// the sums of all chunks' histograms, scanned; what min-p keeps, and the weight of all entries
template <int NT> ME_DEV void load_hist(Shared<NT>& s, const SampleArgs& a, const RowWs& w, uint32_t& n_all, u64& m_all, uint32_t& n_keep, u64& m_keep, u64& m_tot) {
    constexpr int PB = NB / NT;
    const int lane = threadIdx.x & 63;
    n_keep = lane < a.splits ? w.n_keep[lane] : 0;
    m_keep = lane < a.splits ? w.m_keep[lane] : 0;
    m_tot = lane < a.splits ? w.m_tot[lane] : 0;
    uint32_t c[PB] = {};
    u64 m[PB] = {};
    for (int q0 = 0; q0 < a.splits; q0 += 4) {                // loads of four chunks in flight, no branch between them
        uint32_t x[4][PB];
        u64 y[4][PB];
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int i = 0; i < PB; ++i) {
                const int at = min(q0 + q, a.splits - 1) * NB + threadIdx.x + i * NT;
                x[q][i] = w.cnt[at];
                y[q][i] = w.mass[at];
            }
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int i = 0; i < PB; ++i) { c[i] += q0 + q < a.splits ? x[q][i] : 0; m[i] += q0 + q < a.splits ? y[q][i] : 0; }
    }
#pragma unroll
    for (int i = 0; i < PB; ++i) { s.cnt[threadIdx.x + i * NT] = c[i]; s.mass[threadIdx.x + i * NT] = m[i]; }
#pragma unroll
    for (int o = 8; o; o >>= 1) { n_keep += __shfl_xor(n_keep, o); m_keep += __shfl_xor(m_keep, o); m_tot += __shfl_xor(m_tot, o); }   // 16 lanes: MAX_SPLIT
    n_keep = __shfl(n_keep, 0);
    m_keep = __shfl(m_keep, 0);
    m_tot = __shfl(m_tot, 0);
    __syncthreads();
    scan_bins<NT, NB>(s, s.cnt, s.mass, n_all, m_all);
    if (!cuts(a)) { n_keep = n_all; m_keep = m_all; m_tot += m_all; }
}

// ids that may not be picked, inside a chunk from j0 on: one bit each, looked at for entries before `end` only (they are mostly the first ids)
struct Barred { const uint32_t* bits; int end; };
template <int NT> ME_DEV Barred bar_ids(const SampleArgs& a, uint32_t* bits, int j0, int j1) {
    if (a.n_special <= 0) return {nullptr, j0};               // uniform
    for (int i = threadIdx.x; i < (j1 - j0 + 31) / 32 + 1; i += NT) bits[i] = 0;             // bits[0]: how far they go
    __syncthreads();
    for (int i = threadIdx.x; i < a.n_special; i += NT) {
        const int j = a.special[i];
        if (j >= j0 && j < j1) { atomicOr(&bits[1 + ((j - j0) >> 5)], 1u << ((j - j0) & 31)); atomicMax(&bits[0], (uint32_t)(j - j0 + 1)); }
    }
    __syncthreads();
    return {bits + 1, j0 + (int)__builtin_amdgcn_readfirstlane((int)bits[0])};
}
// entries [j0, j1) of a row, once each: NaN -> 0, barred ids -> -inf; f(value, index).  Whole blocks of NT * U behind the barred ids, nearly all
// of a row, are read without a bound and without the look at the bits: about a third of a walk's instructions
template <int NT, int U, typename F> ME_DEV void each_entry(const float* lg, int j0, int j1, const Barred& barred, F&& f) {
    const int tid = threadIdx.x;
    int b0 = j0;                                              // uniform
#pragma clang loop unroll(disable)
    for (int part = 0; part < 2; ++part) {
        const int stop = part ? j1 : min(j1, j0 + (max(barred.end, j0) - j0 + NT * U - 1) / (NT * U) * (NT * U));
        for (; b0 < stop; b0 += NT * U) {
            float x[U];
#pragma unroll
            for (int q = 0; q < U; ++q) x[q] = lg[min(b0 + q * NT + tid, j1 - 1)];
#pragma unroll
            for (int q = 0; q < U; ++q) {
                const int j = b0 + q * NT + tid;
                if (j < j1) {
                    float v = x[q];
                    if (v != v) v = 0.f;
                    if (j < barred.end && ((barred.bits[(j - j0) >> 5] >> ((j - j0) & 31)) & 1u)) v = -INFINITY;
                    f(v, j);
                }
                __builtin_amdgcn_sched_barrier(0);            // the entries' f64 chains stay apart (the waves hide them): few registers
            }
        }
        if (part) break;
        for (; b0 + NT * U <= j1; b0 += NT * U) {
            const float* p = lg + b0;
            float x[U];
#pragma unroll
            for (int q = 0; q < U; ++q) x[q] = p[q * NT + tid];
#pragma unroll
            for (int q = 0; q < U; ++q) {
                f(x[q] != x[q] ? 0.f : x[q], b0 + q * NT + tid);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------------------
// the search over a scanned histogram and the entries that `each(low, high, f)` walks (values in an interval).  by_rank: the mass of the first `rank` entries; else the
// first entry whose cumulative weight exceeds `limit` (its word, its rank, the mass before it).  The histogram holds the entries with
// exponents from y_floor on.
// ---------------------------------------------------------------------------------------------------------
template <int NT, typename EACH>
ME_DEV void search(Shared<NT>& s, const Scale& sc, EACH&& each, double y_floor, uint32_t n_all, u64 m_all, bool by_rank, uint32_t rank, u64 limit, u64& word, uint32_t& at, u64& before) {
    const int tid = threadIdx.x;
    uint32_t* cnt = s.cnt;
    u64* mass = s.mass;
    int nb = NB;
    uint32_t total = n_all, c0 = 0;                           // entries and mass before the window of this level
    u64 mtotal = m_all, m0 = 0;
    u64 hi = 0, lo = 0;
    int shift = 0, level = 0, bin0 = 0;
    uint32_t listed = 0;                                      // entries in s.lw, once the window's fit there
    float v_lo = 0.f, v_hi = 0.f;
    if (tid == 0) { s.found_bin = 0; s.found_rank = 0; s.found_mass = 0; s.found_word = 0xffffffffull; }     // index 0
    __syncthreads();
    // 8 bits of the word's range a level: 1 + 8 levels at most, and the loop ends there whatever it finds
#pragma clang loop unroll(disable)
    for (int turn = 0; turn < 10; ++turn) {
        for (int i = tid; i < nb; i += NT) {
            const uint32_t cb = c0 + cnt[i], ce = c0 + (i + 1 < nb ? cnt[i + 1] : total);
            const u64 mb = m0 + mass[i], me = m0 + (i + 1 < nb ? mass[i + 1] : mtotal);
            if (by_rank ? (cb < rank && rank <= ce) : (mb <= limit && limit < me)) s.found_bin = (uint32_t)i;
        }
        if (tid == 0) s.n_list = 0;
        __syncthreads();
        const int bin = (int)s.found_bin;
        const uint32_t cb = c0 + cnt[bin], n = c0 + (bin + 1 < nb ? cnt[bin + 1] : total) - cb;
        const u64 mb = m0 + mass[bin];
        if (level == 0) bin0 = bin;
        else {                                                // the piece's words; its lower end may lie below zero (words are as small as 2^55)
            const u64 top = hi - ((u64)bin << shift), span = ((u64)1 << shift) - 1;
            lo = max(lo, top > span ? top - span : 0);
            hi = top;
        }
        c0 = cb;
        m0 = mb;
        if (level == 0) sc.interval(bin0, bin0, v_lo, v_hi);
        auto inside = [&](float v, u64 w) { return level == 0 ? sc.bin(v) == bin0 && sc.exponent(v) >= y_floor : w <= hi && w >= lo; };
        const bool collect = listed == 0 && n <= CL;
        if (collect) {
            each(v_lo, v_hi, [&](float v, int j) {
                const u64 w = word_of(v, j);
                if (inside(v, w)) { const uint32_t k = atomicAdd(&s.n_list, 1u); if (k < CL) s.lw[k] = w; }
            });
        }
        __syncthreads();                                      // and found_bin, cnt, mass have been read
        if (collect) listed = min(s.n_list, (uint32_t)CL);
        if ((collect || listed) && n <= NL) {
            if (listed > n) {                                 // the window's part of the list to its front
                const uint32_t per = (listed + NT - 1) / NT;
                u64 mine[CL / NT > 0 ? CL / NT : 1];
#pragma unroll
                for (uint32_t q = 0; q < sizeof(mine) / 8; ++q) { const uint32_t e = tid + q * NT; mine[q] = q < per && e < listed ? s.lw[e] : 0; }
                if (tid == 0) s.n_list = 0;
                __syncthreads();
#pragma unroll
                for (uint32_t q = 0; q < sizeof(mine) / 8; ++q) if (mine[q] && mine[q] <= hi && mine[q] >= lo) s.lw[atomicAdd(&s.n_list, 1u)] = mine[q];
                __syncthreads();
            }
            for (uint32_t e = tid; e < n; e += NT) { const u64 m = sc.weight(sc.exponent(value_of(s.lw[e]))); s.lm[e] = m; s.lc[e] = m; s.lr[e] = 0; }
            __syncthreads();
            // each entry against all others: NT / NL threads share an entry, their sums are whole numbers
            {
                constexpr uint32_t P = NT / NL;
                const uint32_t e = tid % NL, per = (n + P - 1) / P, k0 = (tid / NL) * per, k1 = min(k0 + per, n);
                if (e < n && k0 < k1) {
                    const u64 me = s.lw[e];
                    uint32_t r = 0;
                    u64 cum = 0;
#pragma clang loop unroll_count(4)
                    for (uint32_t k = k0; k < k1; ++k) { const bool ahead = s.lw[k] > me; r += ahead; cum += ahead ? s.lm[k] : 0; }
                    if (r) { atomicAdd(&s.lr[e], r); atomicAdd(&s.lc[e], cum); }
                }
            }
            __syncthreads();
            for (uint32_t e = tid; e < n; e += NT) {
                const u64 cum = m0 + s.lc[e], own = s.lm[e];
                const uint32_t r = c0 + s.lr[e];
                const bool hit = by_rank ? r + 1 == rank : (cum > limit && cum - own <= limit);
                if (hit) { s.found_word = s.lw[e]; s.found_rank = r; s.found_mass = by_rank ? cum : cum - own; }
            }
            break;
        }
        // too many for that: the words between the window's first and last, cut into 256 pieces of their range (words differ, so a
        // few levels end at one entry each); from the list where the window fits there, else from the row
        auto window = [&](auto&& f) {
            if (listed) { for (uint32_t e = tid; e < listed; e += NT) { const u64 w = s.lw[e]; const float v = value_of(w); if (inside(v, w)) f(w); } }
            else each(v_lo, v_hi, [&](float v, int j) { const u64 w = word_of(v, j); if (inside(v, w)) f(w); });
        };
        u64 wmax = 0, wmin = 0;                               // wmin as the maximum of the complement
        window([&](u64 w) { wmax = max(wmax, w); wmin = max(wmin, ~w); });
        for (int i = tid; i < NB1; i += NT) { s.cnt1[i] = 0; s.mass1[i] = 0; }
        block_max64(s, wmax, wmin);
        wmin = ~wmin;
        const int width = 64 - (int)__builtin_clzll((wmax - wmin) | 1);
        const int next = max(0, width - 8);                   // 2^8 = NB1 pieces
        window([&](u64 w) {
            const int i = (int)((wmax - w) >> next);
            const u64 m = sc.weight(sc.exponent(value_of(w)));
            atomicAdd(&s.cnt1[i], 1u);
            if (m) atomicAdd(&s.mass1[i], m);
        });
        __syncthreads();
        hi = wmax;
        lo = wmin;
        shift = next;
        level = 1;
        cnt = s.cnt1;
        mass = s.mass1;
        nb = NB1;
        scan_bins<NT, NB1>(s, cnt, mass, total, mtotal);
    }
    __syncthreads();
    word = s.found_word;
    at = s.found_rank;
    before = s.found_mass;
    __syncthreads();
}

// ---- top-k, then min-p, then the nucleus, then the draw.  n_keep, m_keep: what min-p leaves (with top-k: of the entries in bins up to
//      its border's); m_tot: the weight of all entries (read where top-k does not cut).  searcher(by_rank, rank, limit, word, at, mass)
template <typename S>
ME_DEV void choose(const SampleArgs& a, int b, float u, uint32_t n_keep, u64 m_keep, u64 m_tot, S&& searcher) {
    u64 word = 0, mass = 0, tot = m_tot, tot_k = m_tot, limit = 0;
    uint32_t at = 0, n = (uint32_t)a.V;
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
        searcher(phase == 0, n, limit, word, at, mass);
        if (phase == 0) tot = mass;
        if (phase == 1) { n = at > 0 ? at : 1; tot = at > 0 ? mass : (u64)1 << FRAC; }        // its first entry always stays
    }
    if (threadIdx.x == 0) finish(a, b, index_of(word), (int)n);
}

// ---------------------------------------------------------------------------------------------------------
// rows of up to ONE_BLOCK symbols: one block, the row in LDS.  Without top-k one walk makes the histogram of what min-p keeps.  With
// top-k the walk only counts, and the few entries up to its border's bin are collected; they alone get weights and take the row's place
// in the searches (64 x 32000, top_k 200: 24 us; 32 when the row was walked again for each search).
// ---------------------------------------------------------------------------------------------------------
template <int NT>
__global__ __launch_bounds__(NT) void sample_row_kernel(const SampleArgs a) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    Shared<NT>& s = *reinterpret_cast<Shared<NT>*>(smem);
    u64* head = reinterpret_cast<u64*>(smem + sizeof(Shared<NT>));                    // [SL]
    float* row = reinterpret_cast<float*>(head + SL);
    const int tid = threadIdx.x, b = blockIdx.x, V = a.V;
    const float* lg = a.logits + (size_t)b * a.ld;
    const float temp = row_temp(a, b), u = row_u(a, b);
    constexpr int L = 8;
    for (int j0 = tid; j0 < V; j0 += NT * L) {
        float x[L];
#pragma unroll
        for (int q = 0; q < L; ++q) x[q] = lg[min(j0 + q * NT, V - 1)];
#pragma unroll
        for (int q = 0; q < L; ++q) if (j0 + q * NT < V) row[j0 + q * NT] = x[q] != x[q] ? 0.f : x[q];
    }
    const int V4 = (V + 3) / 4;                               // filled up with entries of weight 0 behind all others
    if (tid < 4 * V4 - V) row[V + tid] = -INFINITY;
    if (tid < 32) s.tab[tid] = exp2(tid * (1.0 / 32));
    for (int i = tid; i < NB; i += NT) { s.cnt[i] = 0; s.mass[i] = 0; }
    __syncthreads();
    for (int i = tid; i < a.n_special; i += NT) { const int j = a.special[i]; if (j >= 0 && j < V) row[j] = -INFINITY; }
    __syncthreads();
    const f32x4_t* row4 = reinterpret_cast<const f32x4_t*>(row);
    float mx = -INFINITY;
    for (int i = tid; i < V4; i += NT) { const f32x4_t x = row4[i]; mx = fmaxf(fmaxf(mx, fmaxf(x[0], x[1])), fmaxf(x[2], x[3])); }
    mx = block_max<NT>(s, mx);
    if (mx == -INFINITY) {                                    // nothing to choose from
        if (tid == 0) finish(a, b, 0, 0);
        return;
    }
    Scale sc;
    sc.set(mx, temp, s.tab);
    auto each = [&](float low, float high, auto&& f) {
        for (int i = tid; i < V4; i += NT) {
            const f32x4_t x = row4[i];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                if (x[q] >= low && x[q] <= high) f(x[q], 4 * i + q);
                __builtin_amdgcn_sched_barrier(0);            // the entries' f64 chains stay apart (the waves hide them): few registers
            }
        }
    };
    uint32_t n_keep = 0, n_all;
    u64 m_keep = 0, m_tot = 0, m_all;
    const double kept = keep_floor(a);
    float v_lo, v_hi;
    uint32_t n_head = 0;                                      // entries in `head`, where they hold all that can be kept
    if (cuts(a)) {
        // counts of all entries; only those in bins up to the one that holds rank top_k can be kept, and only they get a weight
        each(-INFINITY, INFINITY, [&](float v, int) { atomicAdd(&s.cnt[sc.bin(v)], 1u); });
        __syncthreads();
        scan_bins<NT, NB>(s, s.cnt, s.mass, n_all, m_all);
        for (int i = tid; i < NB; i += NT) if (s.cnt[i] < (uint32_t)a.top_k && (uint32_t)a.top_k <= (i + 1 < NB ? s.cnt[i + 1] : n_all)) s.found_bin = (uint32_t)i;
        __syncthreads();
        const int bin_k = (int)s.found_bin;
        n_head = bin_k + 1 < NB ? s.cnt[bin_k + 1] : n_all;
        if (n_head > SL) n_head = 0;
        sc.interval(0, bin_k, v_lo, v_hi);
        auto add = [&](float v, int bin) {
            const double e = sc.exponent(v);
            const u64 w = sc.weight(e);
            const bool keep = e >= kept;
            n_keep += keep;
            m_keep += keep ? w : 0;
            atomicAdd(&s.mass[bin], w);
        };
        if (n_head) {                                         // few: collected first, a thread each from here on
            if (tid == 0) s.n_list = 0;
            __syncthreads();
            each(v_lo, v_hi, [&](float v, int j) { if (sc.bin(v) <= bin_k) head[atomicAdd(&s.n_list, 1u)] = word_of(v, j); });
            __syncthreads();
            for (uint32_t i = tid; i < n_head; i += NT) { const float v = value_of(head[i]); add(v, sc.bin(v)); }
        } else each(v_lo, v_hi, [&](float v, int) { const int bin = sc.bin(v); if (bin <= bin_k) add(v, bin); });
        __syncthreads();
        scan_mass<NT>(s, s.mass, m_all);                      // the counts are scanned already
        block_sum3(s, n_keep, m_keep, m_tot);
    } else {
        // the histogram holds what min-p keeps; what it drops is only read for the sum that the nucleus refers to
        const bool rest = has_nucleus(a) && a.y_min > -INFINITY;
        v_lo = rest || sc.inf ? -INFINITY : (float)fmax((double)mx + kept / sc.c * 1.0001 - 1e-5 * fabs((double)mx), -3.402823466e38);
        each(v_lo, INFINITY, [&](float v, int) {
            const double e = sc.exponent(v);
            const u64 w = sc.weight(e);
            if (e >= kept) {
                const int bin = sc.bin(v);
                atomicAdd(&s.cnt[bin], 1u);
                atomicAdd(&s.mass[bin], w);
            } else if (rest) m_tot += w;
        });
        __syncthreads();
        scan_bins<NT, NB>(s, s.cnt, s.mass, n_all, m_all);
        n_keep = 0;
        if (rest) block_sum3(s, n_keep, m_keep, m_tot);
        n_keep = n_all;
        m_keep = m_all;
        m_tot += m_all;
    }
    choose(a, b, u, n_keep, m_keep, m_tot, [&](bool by_rank, uint32_t rank, u64 limit, u64& word, uint32_t& at, u64& mass) {
        search<NT>(s, sc, [&](float low, float high, auto&& f) {
            if (n_head) { for (uint32_t i = tid; i < n_head; i += NT) { const float v = value_of(head[i]); if (v >= low && v <= high) f(v, index_of(head[i])); } }
            else each(low, high, f);
        }, floor_of(a), n_all, m_all, by_rank, rank, limit, word, at, mass);
    });
}

// ---------------------------------------------------------------------------------------------------------
// wider rows: grid (splits, B) blocks of a chunk each.  Bounded by the histogram's and the gathering's instructions, about 30 an entry
// (128 x 131071: 29 and 21 us; their bytes alone would take 13 us each at the rate of a copy)
// ---------------------------------------------------------------------------------------------------------
constexpr int WT = 512;                                       // threads of a chunk's block
constexpr int PT = 256;                                       // and of the block that finishes a row

__global__ __launch_bounds__(WT) void sample_max_kernel(const SampleArgs a) {
    extern __shared__ uint32_t bits[];
    __shared__ float red[WT / 64];
    const int b = blockIdx.y, j0 = blockIdx.x * a.chunk, j1 = min(j0 + a.chunk, a.V);
    const RowWs w = row_ws(a, b);
    const Barred barred = bar_ids<WT>(a, bits, j0, j1);
    float mx = -INFINITY;
    each_entry<WT, 8>(a.logits + (size_t)b * a.ld, j0, j1, barred, [&](float v, int) { mx = fmaxf(mx, v); });
    mx = wave_max(mx);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = mx;
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
        for (int i = 0; i < WT / 64; ++i) mx = fmaxf(mx, red[i]);
        w.mx[blockIdx.x] = mx;
        if (blockIdx.x == 0) w.n_list[0] = 0;
    }
}
ME_DEV float row_max(const SampleArgs& a, const RowWs& w) {
    const int lane = threadIdx.x & 63;
    return wave_max(lane < a.splits ? w.mx[lane] : -INFINITY);
}

__global__ __launch_bounds__(WT) void sample_hist_kernel(const SampleArgs a) {
    extern __shared__ uint32_t bits[];
    __shared__ Shared<WT> s;
    const int tid = threadIdx.x, b = blockIdx.y, j0 = blockIdx.x * a.chunk, j1 = min(j0 + a.chunk, a.V);
    const RowWs w = row_ws(a, b);
    if (tid < 32) s.tab[tid] = exp2(tid * (1.0 / 32));
    for (int i = tid; i < NB; i += WT) { s.cnt[i] = 0; s.mass[i] = 0; }
    const Barred barred = bar_ids<WT>(a, bits, j0, j1);
    const float mx = row_max(a, w);
    if (mx == -INFINITY) return;                              // the last launch sees it too
    Scale sc;
    sc.set(mx, row_temp(a, b), s.tab);
    __syncthreads();
    uint32_t n_keep = 0;
    u64 m_keep = 0, m_tot = 0;
    const bool minp = a.y_min > -INFINITY;
    const double kept = keep_floor(a);
    const float* lg = a.logits + (size_t)b * a.ld;
    if (cuts(a)) {                                            // with top-k the histogram holds every entry
        each_entry<WT, 8>(lg, j0, j1, barred, [&](float v, int) {
            const double e = sc.exponent(v);
            const u64 m = sc.weight(e);
            const bool keep = e >= kept;
            n_keep += keep;
            m_keep += keep ? m : 0;
            const int bin = sc.bin(v);
            atomicAdd(&s.cnt[bin], 1u);
            atomicAdd(&s.mass[bin], m);
        });
        block_sum3(s, n_keep, m_keep, m_tot);
    } else {                                                  // else what min-p keeps; the rest counts for the nucleus' sum
        const bool rest = minp && has_nucleus(a);
        each_entry<WT, 8>(lg, j0, j1, barred, [&](float v, int) {
            const double e = sc.exponent(v);
            const u64 m = sc.weight(e);
            if (e >= kept) {
                const int bin = sc.bin(v);
                atomicAdd(&s.cnt[bin], 1u);
                atomicAdd(&s.mass[bin], m);
            } else if (rest) m_tot += m;
        });
        if (rest) block_sum3(s, n_keep, m_keep, m_tot);
        else __syncthreads();
    }
    if (tid == 0) { w.n_keep[blockIdx.x] = n_keep; w.m_keep[blockIdx.x] = m_keep; w.m_tot[blockIdx.x] = m_tot; }
    for (int i = tid; i < NB; i += WT) { w.cnt[blockIdx.x * NB + i] = s.cnt[i]; w.mass[blockIdx.x * NB + i] = s.mass[i]; }
}

// the bins that can hold a border, from the histogram alone: each search ends in a known bin, and the mass inside the
// bins of the earlier searches bounds the limits of the later ones.  Up to three ranges of bins.
template <int NT> ME_DEV void border_bins(Shared<NT>& s, const SampleArgs& a, float u, uint32_t n_all, u64 m_all, uint32_t n_keep, u64 m_keep, u64 m_tot, int (&lo)[3], int (&hi)[3]) {
    auto before = [&](int bin) -> u64 { return bin < NB ? s.mass[bin] : m_all; };
    auto find = [&](bool by_rank, uint32_t rank, u64 limit) -> int {
        __syncthreads();
        for (int i = threadIdx.x; i < NB; i += NT) {
            const uint32_t ce = i + 1 < NB ? s.cnt[i + 1] : n_all;
            if (by_rank ? (s.cnt[i] < rank && rank <= ce) : (s.mass[i] <= limit && limit < before(i + 1))) s.found_bin = (uint32_t)i;
        }
        __syncthreads();
        return (int)s.found_bin;
    };
    uint32_t n = (uint32_t)a.V;
    u64 k_lo = m_tot, k_hi = m_tot;
#pragma unroll
    for (int i = 0; i < 3; ++i) { lo[i] = 0; hi[i] = -1; }
    if (a.top_k > 0 && (uint32_t)a.top_k < n) {
        n = (uint32_t)a.top_k;
        lo[0] = hi[0] = find(true, n, 0);
        k_lo = before(lo[0]);
        k_hi = before(lo[0] + 1);
    }
    u64 t_lo = k_lo, t_hi = k_hi;
    if (n_keep < n) t_lo = t_hi = m_keep;
    if (a.top_p > 0.f && a.top_p < 1.f) {
        const u64 l_lo = (u64)((double)a.top_p * (double)k_lo), l_hi = (u64)((double)a.top_p * (double)k_hi);
        if (l_lo < t_hi) {
            lo[1] = find(false, 0, min(l_lo, m_all - 1));
            hi[1] = find(false, 0, min(l_hi, m_all - 1));
            t_lo = min(t_lo, before(lo[1]));
            t_hi = min(t_hi, before(hi[1] + 1));
        }
    }
    t_lo = max(t_lo, (u64)1 << FRAC);                         // the first entry always stays
    t_hi = max(t_hi, t_lo);
    const double uu = u > 0.f ? fmin((double)u, 1.0) : 0.0;
    const u64 d_lo = (u64)(uu * (double)t_lo), d_hi = (u64)(uu * (double)t_hi);
    lo[2] = find(false, 0, min(d_lo - min(d_lo, (u64)1), m_all - 1));
    hi[2] = find(false, 0, min(d_hi, m_all - 1));
}

__global__ __launch_bounds__(WT) void sample_gather_kernel(const SampleArgs a) {
    extern __shared__ uint32_t bits[];
    __shared__ Shared<WT> s;
    __shared__ uint32_t base;
    __shared__ u64 mine[SL];
    const int tid = threadIdx.x, b = blockIdx.y, j0 = blockIdx.x * a.chunk, j1 = min(j0 + a.chunk, a.V);
    const RowWs w = row_ws(a, b);
    const float mx = row_max(a, w);
    if (mx == -INFINITY) return;
    const Barred barred = bar_ids<WT>(a, bits, j0, j1);
    uint32_t n_all, n_keep;
    u64 m_all, m_keep, m_tot;
    load_hist<WT>(s, a, w, n_all, m_all, n_keep, m_keep, m_tot);
    int lo[3], hi[3];
    border_bins<WT>(s, a, row_u(a, b), n_all, m_all, n_keep, m_keep, m_tot, lo, hi);
    if (blockIdx.x == 0 && tid == 0) {
#pragma unroll
        for (int i = 0; i < 3; ++i) { w.ranges[2 * i] = lo[i]; w.ranges[2 * i + 1] = hi[i]; }
    }
    if (tid == 0) s.n_list = 0;
    __syncthreads();
    Scale sc;
    sc.set(mx, row_temp(a, b), s.tab);
    // a chunk's members wait in LDS for one reservation in the row's list; what does not fit there either
    // makes the count exceed GL, and the last launch then reads the row itself
    float v_lo[3], v_hi[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) sc.interval(lo[i], hi[i], v_lo[i], v_hi[i]);
    auto keep = [&](float v, int j) { const uint32_t k = atomicAdd(&s.n_list, 1u); if (k < (uint32_t)SL) mine[k] = word_of(v, j); };
    auto in = [&](float v, int i) { return v >= v_lo[i] && v <= v_hi[i]; };
    const float* lg = a.logits + (size_t)b * a.ld;
    if (cuts(a)) each_entry<WT, 8>(lg, j0, j1, barred, [&](float v, int j) { if (in(v, 0) || in(v, 1) || in(v, 2)) keep(v, j); });
    else each_entry<WT, 8>(lg, j0, j1, barred, [&](float v, int j) { if (in(v, 1) || in(v, 2)) keep(v, j); });
    __syncthreads();
    const uint32_t n = s.n_list;
    if (tid == 0) base = n ? atomicAdd(w.n_list, n > (uint32_t)SL ? (uint32_t)GL + 1 : n) : 0;      // at most MAX_SPLIT of these: no overflow
    __syncthreads();
    if (n > (uint32_t)SL) return;
    for (uint32_t i = tid; i < n; i += WT) if (base + i < (uint32_t)GL) w.list[base + i] = mine[i];
}

template <int NT>
__global__ __launch_bounds__(NT) void sample_pick_kernel(const SampleArgs a) {
    extern __shared__ uint32_t bits[];
    __shared__ Shared<NT> s;
    __shared__ u64 list[GL];
    const int tid = threadIdx.x, b = blockIdx.x;
    const RowWs w = row_ws(a, b);
    const float mx = row_max(a, w);
    if (mx == -INFINITY) {
        if (tid == 0) finish(a, b, 0, 0);
        return;
    }
    const float temp = row_temp(a, b), u = row_u(a, b);
    if (tid < 32) s.tab[tid] = exp2(tid * (1.0 / 32));
    const uint32_t nl = w.n_list[0];
    for (uint32_t i = tid; i < min(nl, (uint32_t)GL); i += NT) list[i] = w.list[i];
    const Barred barred = bar_ids<NT>(a, bits, 0, a.V);
    uint32_t n_all, n_keep;
    u64 m_all, m_keep, m_tot;
    load_hist<NT>(s, a, w, n_all, m_all, n_keep, m_keep, m_tot);
    Scale sc;
    sc.set(mx, temp, s.tab);
    int range[6];
#pragma unroll
    for (int i = 0; i < 6; ++i) range[i] = w.ranges[i];
    choose(a, b, u, n_keep, m_keep, m_tot, [&](bool by_rank, uint32_t rank, u64 limit, u64& word, uint32_t& at, u64& mass) {
        // the bin of this search: gathered, or the whole row is walked
        __syncthreads();
        for (int i = tid; i < NB; i += NT) {
            const uint32_t ce = i + 1 < NB ? s.cnt[i + 1] : n_all;
            const u64 me = i + 1 < NB ? s.mass[i + 1] : m_all;
            if (by_rank ? (s.cnt[i] < rank && rank <= ce) : (s.mass[i] <= limit && limit < me)) s.found_bin = (uint32_t)i;
        }
        __syncthreads();
        const int bin = (int)s.found_bin;
        const bool have = nl <= (uint32_t)GL && ((bin >= range[0] && bin <= range[1]) || (bin >= range[2] && bin <= range[3]) || (bin >= range[4] && bin <= range[5]));
        __syncthreads();
        search<NT>(s, sc, [&](float low, float high, auto&& f) {
            if (have) { for (uint32_t i = tid; i < nl; i += NT) { const float v = value_of(list[i]); if (v >= low && v <= high) f(v, index_of(list[i])); } }
            else each_entry<NT, 4>(a.logits + (size_t)b * a.ld, 0, a.V, barred, [&](float v, int j) { if (v >= low && v <= high) f(v, j); });
        }, floor_of(a), n_all, m_all, by_rank, rank, limit, word, at, mass);
    });
}

// allows a kernel more than 64 KB of LDS, once per device
template <typename K> bool allow_lds(K kernel, size_t bytes, size_t fixed, bool (&done)[64]) {
    if (bytes <= 65536) return true;
    int dev = 0;
    (void)hipGetDevice(&dev);
    if (dev >= 0 && dev < 64 && done[dev]) return true;
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024 - (int)fixed) != hipSuccess) return false;
    if (dev >= 0 && dev < 64) done[dev] = true;
    return true;
}

// chunks of a wide row: two blocks for each CU over the batch, 2048 symbols a chunk at least
int splits_of(int B, int V) { return std::max(1, std::min(std::min(512 / std::max(B, 1), (V + 2047) / 2048), MAX_SPLIT)); }

// the least exponent whose weight, rounded to 64 bits, reaches min_p: half a step of the 64 bits below 1 (all that are 1 in 64 bits pass a min_p of 1)
double least_exponent(float min_p) { return log2((double)min_p) - 0x1p-54 * 1.4426950408889634074; }

int sample_call(SampleArgs& a, int B, void* ws, size_t ws_bytes, hipStream_t st) {
    static bool big1[64] = {}, big2[64] = {};
    if (a.V <= ONE_BLOCK) {
        // 256 threads to 2048 symbols: fewer waves meet at each barrier (2048 symbols on 256 / 2049 on 1024 threads: 4 rows 8.6 / 10.6 us, 64: 10.5 / 11.2)
        if (a.V <= 2048) sample_row_kernel<256><<<B, 256, sizeof(Shared<256>) + SL * 8 + (size_t)(a.V + 3) / 4 * 16, st>>>(a);
        else {
            static_assert(sizeof(Shared<1024>) + SL * 8 + (size_t)ONE_BLOCK * 4 <= 160 * 1024, "the widest row of one block");
            const size_t lds = sizeof(Shared<1024>) + SL * 8 + (size_t)(a.V + 3) / 4 * 16;
            if (!allow_lds(&sample_row_kernel<1024>, lds, 0, big1)) return ME_ERR_LAUNCH;
            sample_row_kernel<1024><<<B, 1024, lds, st>>>(a);
        }
        return me_launch_status();
    }
    a.splits = splits_of(B, a.V);
    a.chunk = (a.V + a.splits - 1) / a.splits;
    if (!ws || ((uintptr_t)ws & 15) || ws_bytes < (size_t)B * row_ws_bytes(a.splits)) return ME_ERR_WORKSPACE;
    a.ws = (char*)ws;
    static_assert(sizeof(Shared<WT>) + SL * 8 + 16 + ME_SAMPLE_MAX_VOCAB / 8 + 8 <= 65536, "a chunk of the widest row, with its barred ids");
    const dim3 grid(a.splits, B);
    const size_t bits = a.n_special > 0 ? (size_t)(a.chunk + 31) / 32 * 4 + 4 : 0, all = a.n_special > 0 ? (size_t)(a.V + 31) / 32 * 4 + 4 : 0;
    if (!allow_lds(&sample_pick_kernel<PT>, sizeof(Shared<PT>) + GL * 8 + all, sizeof(Shared<PT>) + GL * 8 + 64, big2)) return ME_ERR_LAUNCH;
    sample_max_kernel<<<grid, WT, bits, st>>>(a);
    sample_hist_kernel<<<grid, WT, bits, st>>>(a);
    sample_gather_kernel<<<grid, WT, bits, st>>>(a);
    sample_pick_kernel<PT><<<B, PT, all, st>>>(a);
    return me_launch_status();
}

}  // namespace

size_t me_sample_ws_bytes(int B, int V) { return B > 0 && V > ONE_BLOCK && V <= ME_SAMPLE_MAX_VOCAB ? (size_t)B * row_ws_bytes(splits_of(B, V)) : 0; }

extern "C" {

int me_sample_minp(const float* logits, int ld, int V, const int32_t* special, int n_special, const float* temp, int top_k, float top_p,
                   float min_p, const float* u, int64_t* out_ids, int32_t* n_choices, int B, void* ws, size_t ws_bytes, void* stream) {
    me_clear_error();
    if (!logits || !temp || !u || !out_ids || (n_special > 0 && !special)) return ME_ERR_NULL;
    if (B < 0 || B > 65535 || V <= 0 || V > ME_SAMPLE_MAX_VOCAB || ld < V || n_special < 0 || !(min_p >= 0.f && min_p <= 1.f)) return ME_ERR_BAD_SHAPE;
    if (B == 0) return ME_OK;
    SampleArgs a = {};
    a.logits = logits; a.ld = ld; a.V = V; a.special = special; a.n_special = n_special; a.temp = temp; a.top_k = top_k; a.top_p = top_p;
    a.y_min = least_exponent(min_p); a.u = u; a.out = out_ids; a.choices = n_choices;
    return sample_call(a, B, ws, ws_bytes, (hipStream_t)stream);
}

int me_sample_minp_step(const float* logits, int ld, int V, const int32_t* special, int n_special, const int64_t* prev_tok,
                        const uint8_t* is_timeshift, float* repeat_counts, float temp_note, float temp_rest, float penalty_coeff, int top_k,
                        float top_p, float min_p, const float* u_table, int u_ld, const int32_t* pos, int pos0, int64_t* out_ids,
                        int32_t* n_choices, int B, void* ws, size_t ws_bytes, void* stream) {
    me_clear_error();
    if (!logits || !prev_tok || !is_timeshift || !repeat_counts || !u_table || !pos || !out_ids || (n_special > 0 && !special)) return ME_ERR_NULL;
    if (B < 0 || B > 65535 || V <= 0 || V > ME_SAMPLE_MAX_VOCAB || ld < V || u_ld < B || n_special < 0 || !(min_p >= 0.f && min_p <= 1.f)) return ME_ERR_BAD_SHAPE;
    if (B == 0) return ME_OK;
    SampleArgs a = {};
    a.logits = logits; a.ld = ld; a.V = V; a.special = special; a.n_special = n_special; a.top_k = top_k; a.top_p = top_p;
    a.y_min = least_exponent(min_p); a.u = u_table; a.out = out_ids; a.choices = n_choices;
    a.prev = prev_tok; a.is_timeshift = is_timeshift; a.repeats = repeat_counts; a.pos = pos; a.pos0 = pos0; a.u_ld = u_ld;
    a.temp_note = temp_note; a.temp_rest = temp_rest; a.penalty = penalty_coeff;
    return sample_call(a, B, ws, ws_bytes, (hipStream_t)stream);
}

}  // extern "C"
