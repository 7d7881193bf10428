// Sampling the next token from rows of logits (omg_dev_sample).
//
// A filter keeps the first n tokens in the order (z descending, index
// ascending), so a cut is one item (z's key, index): what comes before it
// stays.  Masses are whole numbers W(z) = round(2^42 exp((z - max) / T)),
// at most 2^20 of them: they add up to the same in any order, so neither
// atomics nor the split of a row over threads leave a trace in the result.
// exp is taken in 64 bits: a token's border in the running mass is met by a
// random number closer than f32's error in one row of a few hundred.
//
// Rows of up to 32,768 logits take one workgroup each (sample_short), which
// reads them once from memory and again from its L2.  Longer rows are read
// once by the whole chip (sample_stats: per 2,048 logits the maximum, its
// index and, where the row's filters need it, the sum of exp; per 16 the
// maximum), then one workgroup a row finishes (sample_long).  Both look for a
// threshold that few logits pass but all that can be kept do, from the
// maxima of groups of 16: the k-th largest of these maxima has k logits at or
// above it; min_p's threshold is its own; for top_p alone a guess is taken
// and proved by the mass above it.  The logits above it are gathered into a
// list in LDS, where the exact cuts and the drawn token are found by
// comparing all pairs (up to 256) or by histograms over the items' digits.
// Where the kept tokens do not fit the list, the row's masses are summed by
// bins of their distance from the maximum, which leaves one bin's logits to
// order exactly, and the kept masses by segments in index order: by the
// row's workgroup, or for long rows by the whole chip (sample_bins,
// sample_draw).
//
// The code of a pass is kept short (rolled loops over memory, not a row in
// registers): a workgroup that runs through it once waits for instructions
// more than for data; a row of 25,000 held in 32 registers a thread took 14.5
// us for its maximum alone, and 14 more for each unrolled pass of exp.
#include <algorithm>
#include <string>

#include "common.h"
#include "kern_common.h"
#include "paged.h"

namespace omg {

namespace {

constexpr int NT = 1024;          // threads of a row's workgroup
constexpr int NWAVE = NT / WAVE;
constexpr int CHUNK = 2048;       // logits of a wave of sample_stats
constexpr int GROUP = 16;         // logits of a group maximum there
constexpr int CAP = 8192;         // items of the list
constexpr int BINS = 2048;
constexpr int PAIRS = NT / 4;     // items compared pair by pair: four threads each
constexpr int SEG = 256;          // consecutive logits a wave takes at once
constexpr int64_t SHORT = 32 * NT;  // logits of a row that one workgroup takes alone
constexpr int IDX_BITS = 20;      // vocab <= 2^20
constexpr uint32_t IDX_MASK = (1u << IDX_BITS) - 1;
constexpr double ONE = 4398046511104.0;  // 2^42

// A logit as it is ordered: masked ones (-infinity, NaN) -infinity, -0 the 0 it equals.
__device__ inline float clean(float z) { return z > -INFINITY ? z + 0.0f : -INFINITY; }
// Order-preserving bits of a clean logit; 0 for masked ones.
__device__ inline uint32_t key_of(float z) {
    const uint32_t u = __builtin_bit_cast(uint32_t, z);
    return z == -INFINITY ? 0 : u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ inline float value_of(uint32_t k) {
    return __builtin_bit_cast(float, k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
// An item: larger comes first.
__device__ inline uint64_t item_of(float z, uint32_t i) {
    return uint64_t(key_of(z)) << IDX_BITS | (IDX_MASK - i);
}
__device__ inline float item_value(uint64_t it) { return value_of(uint32_t(it >> IDX_BITS)); }
__device__ inline uint32_t item_index(uint64_t it) { return IDX_MASK - (uint32_t(it) & IDX_MASK); }

// exp((z - max) / T) of a clean logit: 1 at the maximum, whatever it is, 0
// where it is masked.  With t = (z - max) log2(e) / T = n + f, |f| <= 1/2:
// the series of 2^f = exp(f ln 2) to the 11th power (its rest is below
// 2^-46), its exponent raised by n.
struct Weigh {
    double max, inv_t;
    __device__ double operator()(float z) const {
        constexpr double WHOLE = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to a whole number
        double t = (double(z) - max) * (inv_t * 1.4426950408889634);
        t = fmax(t, -1000.0);  // (and NaN, from -infinity / infinity, to -1000)
        const double shifted = t + WHOLE, f = t - (shifted - WHOLE);
        constexpr double L = 0.69314718055994531;
        constexpr double c2 = L * L / 2, c3 = c2 * L / 3, c4 = c3 * L / 4, c5 = c4 * L / 5, c6 = c5 * L / 6,
                         c7 = c6 * L / 7, c8 = c7 * L / 8, c9 = c8 * L / 9, c10 = c9 * L / 10, c11 = c10 * L / 11;
        double p = c11;
        p = fma(p, f, c10);
        p = fma(p, f, c9);
        p = fma(p, f, c8);
        p = fma(p, f, c7);
        p = fma(p, f, c6);
        p = fma(p, f, c5);
        p = fma(p, f, c4);
        p = fma(p, f, c3);
        p = fma(p, f, c2);
        p = fma(p, f, L);
        p = fma(p, f, 1.0);
        const uint64_t n = __builtin_bit_cast(uint64_t, shifted);  // (its low bits: n)
        const double w = __builtin_bit_cast(double, __builtin_bit_cast(uint64_t, p) + (n << 52));
        // an infinite maximum leaves NaN and 2^-1000 above: its equals weigh 1
        return max < INFINITY ? w : z < INFINITY ? 0.0 : 1.0;
    }
    __device__ uint64_t mass(float z) const { return fixed((*this)(z)); }
    // (2^52 + v rounds v to a whole number in its low bits)
    static __device__ uint64_t fixed(double w) {
        return __builtin_bit_cast(uint64_t, fma(w, ONE, 4503599627370496.0)) & 0xfffffffffffffull;
    }
};

// A row's settings; filters that are off have their neutral value.
struct Settings {
    bool greedy;
    int64_t k;      // 0: off
    float p;        // >= 1: off
    double least;   // 0: off
    double inv_t;
    float t;
    __device__ bool need_sum() const { return !greedy && k == 0 && (p < 1.0f || least == 0.0); }
};
__device__ inline Settings settings_of(const SampleArgs& a, int64_t r) {
    Settings s;
    s.t = a.temperature ? a.temperature[r] : 1.0f;
    s.greedy = !(s.t > 0.0f);
    s.inv_t = s.greedy ? 0.0 : 1.0 / double(s.t);
    const int64_t k = a.top_k ? int64_t(a.top_k[r]) : 0;
    s.k = k > 0 && k < a.vocab ? k : 0;
    const float p = a.top_p ? a.top_p[r] : 1.0f;
    s.p = p < 1.0f ? p : 1.0f;
    const float m = a.min_p ? a.min_p[r] : 0.0f;
    s.least = m > 0.0f ? (m < 1.0f ? double(m) : 1.0) : 0.0;
    return s;
}

__device__ inline uint64_t wave_sum_u64(uint64_t v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, WAVE);
    return v;
}
__device__ inline uint64_t wave_scan_u64(uint64_t v, int lane) {  // inclusive
#pragma unroll
    for (int o = 1; o < WAVE; o <<= 1) {
        const uint64_t x = __shfl_up(v, o, WAVE);
        if (lane >= o) v += x;
    }
    return v;
}

struct Shared {
    uint64_t item[CAP];   // the list; without one, the masses of the row's segments
    uint64_t mass[CAP];   // (top bit: under min_p)
    uint64_t hist[BINS];
    uint64_t part[NWAVE];
    uint64_t before, in_bin, total;
    uint32_t bin, kmax, kfirst;
    int count;
};
constexpr uint64_t UNDER = uint64_t(1) << 63;

__device__ inline uint64_t block_sum(uint64_t v, Shared& sm) {
    v = wave_sum_u64(v);
    __syncthreads();
    if (threadIdx.x % WAVE == 0) sm.part[threadIdx.x / WAVE] = v;
    __syncthreads();
    uint64_t s = 0;
#pragma unroll
    for (int i = 0; i < NWAVE; ++i) s += sm.part[i];
    return s;
}

// The bin at which the running sum over h[0 .. n), in ascending or (DOWN)
// descending order, first reaches `target`; the last one in order if it
// never does.  Sets sm.bin, sm.before (the sum before it), sm.in_bin and
// sm.total.
template <bool DOWN>
__device__ inline void pick(const uint64_t* h, int n, uint64_t target, Shared& sm) {
    const int tid = int(threadIdx.x), lane = tid % WAVE, wave = tid / WAVE;
    const int per = (n + NT - 1) / NT;
    __syncthreads();
    uint64_t own = 0;
    for (int i = 0; i < per; ++i) {
        const int j = tid * per + i;
        if (j < n) own += h[DOWN ? n - 1 - j : j];
    }
    const uint64_t scan = wave_scan_u64(own, lane);
    if (lane == WAVE - 1) sm.part[wave] = scan;
    __syncthreads();
    uint64_t base = 0, total = 0;
#pragma unroll
    for (int i = 0; i < NWAVE; ++i) {
        if (i < wave) base += sm.part[i];
        total += sm.part[i];
    }
    uint64_t run = base + scan - own;
    const bool never = total < target;
    if (tid == 0) sm.total = total;
    for (int i = 0; i < per; ++i) {
        const int j = tid * per + i;
        if (j >= n) break;
        const uint64_t x = h[DOWN ? n - 1 - j : j];
        if (never ? j == n - 1 : run < target && run + x >= target) {
            sm.bin = uint32_t(DOWN ? n - 1 - j : j);
            sm.before = run;
            sm.in_bin = x;
        }
        run += x;
    }
    __syncthreads();
}

__device__ inline void clear(uint64_t* h, int n) {
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += NT) h[i] = 0;
    __syncthreads();
}
__device__ inline void add(uint64_t* h, uint64_t v) {
    atomicAdd(reinterpret_cast<unsigned long long*>(h), static_cast<unsigned long long>(v));
}

// The item at which the running share, over the items >= limit from the
// first on, first reaches `target` (>= 1); an item that takes in all of them
// if it never does.  src(f) calls f(item, i) for the thread's items;
// share(item, i) is an item's count or mass.
template <typename S, typename F>
__device__ uint64_t find_cut(S&& src, Shared& sm, uint64_t target, uint64_t limit, F&& share) {
    uint64_t prefix = 0, before = 0;
    int shift = 52;
#pragma unroll 1
    for (int level = 0; level < 5; ++level) {
        const int bits = level < 2 ? 11 : 10;
        shift -= bits;
        clear(sm.hist, 1 << bits);
        src([&](uint64_t it, int i) {
            if (it < limit || (it >> (shift + bits)) != prefix) return;
            const uint64_t v = share(it, i);
            if (v) add(&sm.hist[(it >> shift) & ((1u << bits) - 1)], v);
        });
        pick<true>(sm.hist, 1 << bits, target - before, sm);
        prefix = prefix << bits | sm.bin;
        before += sm.before;
        if (before + sm.in_bin <= target) break;  // the whole bin stays
    }
    const uint64_t cut = prefix << shift;
    return cut > limit ? cut : limit;
}

// Counts of group maxima by their distance from the row's maximum, in bins
// of T / 64 or 1/32, whichever is narrower.  A threshold is a bin's far edge
// (with a slack for the rounding of the bins).
struct Scale {
    float max, per;  // bins per unit of z
    bool whole;      // what lies past the last bin has no mass
    __device__ Scale(float m, float t) : max(m) {
        const float f = 64.0f / t;
        per = f > 32.0f ? (f < 1e30f ? f : 1e30f) : 32.0f;
        whole = float(BINS - 1) > 30.5f * t * per;  // e^-29.9 < 2^-43
    }
    __device__ int bin(float z) const {
        const float x = (max - z) * per;
        return x < float(BINS - 1) ? int(x) : BINS - 1;  // (NaN, infinity - infinity: the last)
    }
};

// A row that is worked on as a whole: each(f) calls f(z, index) for the
// thread's logits, sums(out, m) leaves the sums of m(z, index) over segments
// of SEG.
template <typename T>
struct Row {
    const T* p;
    int64_t n;
    bool wide;  // four elements at once are aligned
    __device__ Row(const T* row, int64_t vocab)
        : p(row), n(vocab), wide(reinterpret_cast<uintptr_t>(row) % (4 * sizeof(T)) == 0 && vocab >= 4) {}
    // The four logits from i (a multiple of 4) on, masked behind the row, in
    // two steps, so that a caller's loads can be under way together.
    typedef T vec __attribute__((ext_vector_type(4)));
    __device__ vec load(int64_t i) const {
        if (wide) return *reinterpret_cast<const vec*>(p + (i + 4 <= n ? i : 0));
        vec v;
#pragma unroll
        for (int c = 0; c < 4; ++c) v[c] = p[i + c < n ? i + c : 0];
        return v;
    }
    __device__ void four(vec v, int64_t i, float* z) const {
        if (i < n && i + 4 > n) {
#pragma unroll
            for (int c = 0; c < 3; ++c) v[c] = p[i + c < n ? i + c : 0];
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) z[c] = i + c < n ? clean(float(v[c])) : -INFINITY;
    }
    // f(z, i) for the four logits z of each of the thread's turns, the next
    // two turns' loads under way; every thread makes the same turns.
    template <typename F>
    __device__ void turns(F&& f) const {
        int64_t i = int64_t(threadIdx.x) * 4;
        vec v0 = load(i), v1 = load(i + NT * 4);
#pragma unroll 1
        for (int64_t base = 0; base < n; base += NT * 8, i += NT * 8) {
            const vec w0 = load(i + NT * 8), w1 = load(i + NT * 12);
            float z[4];
            four(v0, i, z);
            f(z, i);
            four(v1, i + NT * 4, z);
            f(z, i + NT * 4);
            v0 = w0, v1 = w1;
        }
    }
    template <typename F>
    __device__ void each(F&& f) const {
        turns([&](const float* z, int64_t i) {
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (z[c] != -INFINITY) f(z[c], uint32_t(i + c));
        });
    }
    __device__ int segments() const { return int((n + SEG - 1) / SEG); }
    template <typename F>
    __device__ void sums(uint64_t* out, F&& m) const {
        turns([&](const float* z, int64_t i) {
            uint64_t v = 0;
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (z[c] != -INFINITY) v += m(z[c], uint32_t(i + c));
            v = wave_sum_u64(v);
            if (threadIdx.x % WAVE == 0 && i < n) out[i / SEG] = v;
        });
    }
};

struct Result {
    int32_t* token;
    float* logprob;
    Weigh w;
    __device__ void certain(uint32_t i) const {
        *token = int32_t(i);
        if (logprob) *logprob = 0.0f;
    }
    __device__ void write(float z, uint32_t i, uint64_t total) const {
        *token = int32_t(i);
        const double d = double(z) - w.max;
        if (logprob) *logprob = float((d < 0.0 ? d * w.inv_t : 0.0) - log(double(total) / ONE));
    }
};

// The first running mass that exceeds u * total.
__device__ inline uint64_t goal(float u, uint64_t total) {
    const double t = (u > 0.0f ? (u < 1.0f ? double(u) : 1.0) : 0.0) * double(total);
    const uint64_t g = uint64_t(t) + 1;
    return g < total ? g : total;
}
// top_p's: the running mass at which p * total is reached.
__device__ inline uint64_t share_of(float p, uint64_t total) {
    const double t = ceil(double(p) * double(total));
    const uint64_t g = t < 1.0 ? 1 : uint64_t(t);
    return g < total ? g : total;
}

// The drawn logit of one segment: `target` into the masses m(z, i) of its
// logits (its last with a mass where rounding leaves them short of it).
template <typename T, typename F>
__device__ inline void draw_in(const T* p, int64_t n, int64_t first, int count, uint64_t target, uint64_t total,
                               const Result& out, F&& m) {
    if (threadIdx.x >= WAVE) return;
    const int lane = int(threadIdx.x);
    uint64_t run = 0;
    float drawn = 0.0f;
    int64_t index = -1;
    for (int at = 0; at < count; at += WAVE) {
        const int64_t i = first + at + lane;
        const float z = at + lane < count && i < n ? clean(float(p[i])) : -INFINITY;
        const uint64_t v = z != -INFINITY ? m(z, uint32_t(i)) : 0;
        const uint64_t scan = run + wave_scan_u64(v, lane);
        const uint64_t some = __ballot(v > 0), hit = __ballot(v > 0 && scan >= target);
        if (some) {
            const int l = hit ? __builtin_ctzll(hit) : 63 - __builtin_clzll(some);
            drawn = __shfl(z, l, WAVE);
            index = first + at + l;
        }
        if (hit) break;
        run = __shfl(scan, WAVE - 1, WAVE);
    }
    if (lane == 0 && index >= 0) out.write(drawn, uint32_t(index), total);
}

// The exact cuts and the draw over the list's n items (every item that can
// be kept is there); `row_mass`: the mass that top_p is a share of, unless
// top_k is on.
__device__ void finish_list(int n, const Settings& s, float u, uint64_t row_mass, Shared& sm, const Result& out) {
    const Weigh& w = out.w;
    const int tid = int(threadIdx.x);
    __syncthreads();
    for (int i = tid; i < n; i += NT) {
        const double x = w(item_value(sm.item[i]));
        sm.mass[i] = Weigh::fixed(x) | (x >= s.least ? 0 : UNDER);
    }
    __syncthreads();
    if (n <= PAIRS) {
        // Four threads an item: its place, the mass before it; the mass of
        // what stays; the running mass in index order.
        const int e = tid / 4, part = tid % 4;
        const uint64_t mine = e < n ? sm.item[e] : 0, mass = e < n ? sm.mass[e] : 0;
        uint64_t place = 0, before = 0, all = 0;
        for (int j = part; j < n; j += 4) {
            const bool first = sm.item[j] > mine;
            place += first;
            if (first) before += sm.mass[j] & ~UNDER;
        }
        place += __shfl_xor(place, 1, WAVE), before += __shfl_xor(before, 1, WAVE);
        place += __shfl_xor(place, 2, WAVE), before += __shfl_xor(before, 2, WAVE);
        bool keep = e < n && (s.k == 0 || place < uint64_t(s.k));
        if (s.p < 1.0f) {
            all = row_mass;
            if (s.k) all = block_sum(part == 0 && keep ? mass & ~UNDER : 0, sm);
            keep = keep && before < share_of(s.p, all);
        }
        keep = keep && !(mass & UNDER);
        __syncthreads();
        if (part == 0 && e < n) sm.hist[e] = keep ? mass : 0;
        __syncthreads();
        uint64_t run = 0, total = 0;
        const uint32_t at = item_index(mine);
        for (int j = part; j < n; j += 4) {
            const uint64_t m = sm.hist[j];
            total += m;
            if (item_index(sm.item[j]) <= at) run += m;
        }
        run += __shfl_xor(run, 1, WAVE), total += __shfl_xor(total, 1, WAVE);
        run += __shfl_xor(run, 2, WAVE), total += __shfl_xor(total, 2, WAVE);
        const uint64_t target = goal(u, total);
        if (part == 0 && keep && mass > 0 && run >= target && run - mass < target)
            out.write(item_value(mine), at, total);
        return;
    }
    auto items = [&](auto&& f) {
        for (int i = tid; i < n; i += NT) f(sm.item[i], i);
    };
    uint64_t cut = 1;
    if (s.k) cut = find_cut(items, sm, uint64_t(s.k), cut, [](uint64_t, int) { return uint64_t(1); });
    if (s.p < 1.0f) {
        uint64_t all = row_mass;
        if (s.k) {
            uint64_t own = 0;
            items([&](uint64_t it, int i) { own += it >= cut ? sm.mass[i] & ~UNDER : 0; });
            all = block_sum(own, sm);
        }
        cut = find_cut(items, sm, share_of(s.p, all), cut, [&](uint64_t, int i) { return sm.mass[i] & ~UNDER; });
    }
    // the draw: the digits of the index, 10 and 10 bits
    uint64_t own = 0;
    items([&](uint64_t it, int i) { own += it >= cut && !(sm.mass[i] & UNDER) ? sm.mass[i] : 0; });
    const uint64_t total = block_sum(own, sm);
    uint64_t target = goal(u, total);
    uint32_t high = 0;
    for (int level = 0; level < 2; ++level) {
        clear(sm.hist, 1024);
        items([&](uint64_t it, int i) {
            const uint32_t at = item_index(it);
            if (it < cut || (sm.mass[i] & UNDER) || sm.mass[i] == 0 || (level == 1 && at >> 10 != high)) return;
            add(&sm.hist[level == 0 ? at >> 10 : at & 1023], sm.mass[i]);
        });
        pick<false>(sm.hist, 1024, target, sm);
        target -= sm.before;
        if (level == 0) high = sm.bin;
    }
    const uint32_t at = high << 10 | sm.bin;
    items([&](uint64_t it, int) {
        if (item_index(it) == at) out.write(item_value(it), at, total);
    });
}

// The logits of the groups of GROUP whose maxima reach bin `last`: the
// groups' numbers are collected first, so that four threads a group read
// them, two groups at a time in flight.
template <typename T, typename F>
__device__ inline void each_of_groups(const Row<T>& row, const float* groups, const Scale& sc, int last, Shared& sm,
                                      F&& f) {
    uint32_t* ids = reinterpret_cast<uint32_t*>(sm.mass);
    constexpr int MOST = int(sizeof(sm.mass) / 4);  // (a row has up to 2^16 groups)
    const int ngroup = int((row.n + GROUP - 1) / GROUP);
#pragma unroll 1
    for (int g0 = 0; g0 < ngroup; g0 += MOST) {
        const int g1 = g0 + MOST < ngroup ? g0 + MOST : ngroup;
        __syncthreads();
        if (threadIdx.x == 0) sm.bin = 0;
        __syncthreads();
        const int lane = int(threadIdx.x) % WAVE;
        for (int g = g0 + int(threadIdx.x); g - lane < g1; g += NT) {
            const float m = g < g1 ? groups[g] : -INFINITY;
            const bool in = m != -INFINITY && sc.bin(m) <= last;
            const uint64_t some = __ballot(in);
            uint32_t at = 0;
            if (lane == 0 && some) at = atomicAdd(&sm.bin, uint32_t(__popcll(some)));
            at = __builtin_amdgcn_readfirstlane(at);
            if (in) ids[at + __popcll(some & ((uint64_t(1) << lane) - 1))] = uint32_t(g);
        }
        __syncthreads();
        const int count = int(sm.bin);
#pragma unroll 1
        for (int k = int(threadIdx.x) / 4; k < count; k += NT / 2) {
            const int k2 = k + NT / 4;
            const int64_t i0 = int64_t(ids[k]) * GROUP + threadIdx.x % 4 * 4;
            const int64_t i1 = k2 < count ? int64_t(ids[k2]) * GROUP + threadIdx.x % 4 * 4 : row.n;
            const auto v0 = row.load(i0), v1 = row.load(i1);
            float z[8];
            row.four(v0, i0, z);
            row.four(v1, i1, z + 4);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                if (z[c] != -INFINITY) f(z[c], uint32_t(i0 + c));
                if (z[4 + c] != -INFINITY) f(z[4 + c], uint32_t(i1 + c));
            }
        }
    }
    __syncthreads();
}

// Gathers into the list the row's logits that lie in bins 0 .. last.  The
// count may pass CAP: then the list does not hold them all.
template <typename T>
__device__ inline int gather(const Row<T>& row, const float* groups, const Scale& sc, int last, Shared& sm) {
    __syncthreads();
    if (threadIdx.x == 0) sm.count = 0;
    __syncthreads();
    each_of_groups(row, groups, sc, last, sm, [&](float z, uint32_t i) {
        if (sc.bin(z) <= last) {
            const int at = atomicAdd(&sm.count, 1);
            if (at < CAP) sm.item[at] = item_of(z, i);
        }
    });
    return sm.count;
}

// The list that holds every token that the filters can keep, if one can be
// had: its length, or -1.  groups: the maxima of the row's groups.
template <typename T>
__device__ int make_list(const Settings& s, const Scale& sc, Shared& sm, uint64_t row_mass, const Row<T>& row,
                         const float* groups, const Weigh& w) {
    if (!(sc.max < INFINITY)) return -1;
    const bool by_p = s.k == 0 && s.least == 0.0;
    if (s.k || by_p) {
        clear(sm.hist, BINS);
        const int ngroup = int((row.n + GROUP - 1) / GROUP);
#pragma unroll 4
        for (int g = threadIdx.x; g < ngroup; g += NT) {
            const float m = groups[g];
            if (m != -INFINITY) add(&sm.hist[sc.bin(m)], 1);
        }
    }
    // top_p alone: the groups that hold some 100 tokens, then some 4,000
    const uint64_t want = by_p ? share_of(s.p, row_mass) : 0;
#pragma unroll 1
    for (int guess = 0; guess < 2; ++guess) {
        int last;
        if (s.k || by_p) {
            pick<false>(sm.hist, BINS, s.k ? uint64_t(s.k) : guess == 0 ? 96 : 3072, sm);
            last = int(sm.bin);
            if (last == BINS - 1) {
                if (!sc.whole) return -1;
                last = BINS - 2;  // (all that have a mass)
            }
        } else {
            // z >= max + T log(min_p), and a bin to spare
            const float far = float(-log(s.least) * double(s.t)) * sc.per + 1.0f;
            last = far < float(BINS - 2) ? int(far) + 1 : BINS - 1;
            if (last == BINS - 1) return -1;
        }
        const int n = gather(row, groups, sc, last, sm);
        if (n > CAP) return -1;
        if (!by_p) return n;
        uint64_t own = 0;
        for (int i = threadIdx.x; i < n; i += NT) own += w.mass(item_value(sm.item[i]));
        if (block_sum(own, sm) >= want) return n;
    }
    return -1;
}

// The cut over a whole row, found from the sums of `share` by bins of the
// distance from the maximum (in sm.hist): the first items at which the
// running share reaches `target` lie in one bin, whose items are gathered and
// ordered.
template <typename T, typename F>
__device__ uint64_t cut_by_bins(const Row<T>& row, const Scale& sc, Shared& sm, uint64_t target, F&& share) {
    pick<false>(sm.hist, BINS, target, sm);
    const int bin = int(sm.bin);
    const uint64_t left = target - sm.before;
    __syncthreads();
    if (threadIdx.x == 0) sm.count = 0;
    __syncthreads();
    row.each([&](float z, uint32_t i) {
        if (sc.bin(z) == bin) {
            const int at = atomicAdd(&sm.count, 1);
            if (at < CAP) sm.item[at] = item_of(z, i);
        }
    });
    __syncthreads();
    const int n = sm.count;
    if (n <= CAP) {
        auto items = [&](auto&& f) {
            for (int i = threadIdx.x; i < n; i += NT) f(sm.item[i], i);
        };
        const uint64_t edge = find_cut(items, sm, left, 1, [&](uint64_t it, int) { return share(item_value(it)); });
        // (the edge may lie below the bin: the last item of the bin above it)
        __syncthreads();
        if (threadIdx.x == 0) sm.before = ~uint64_t(0);
        __syncthreads();
        items([&](uint64_t it, int) {
            if (it >= edge) atomicMin(reinterpret_cast<unsigned long long*>(&sm.before), static_cast<unsigned long long>(it));
        });
        __syncthreads();
        const uint64_t cut = sm.before;
        __syncthreads();
        return cut == ~uint64_t(0) ? 1 : cut;  // (nothing in the last bin: all stay)
    }
    auto items = [&](auto&& f) { row.each([&](float z, uint32_t i) { f(item_of(z, i), 0); }); };
    return find_cut(items, sm, target, 1, [&](uint64_t it, int) { return share(item_value(it)); });
}

// The exact cuts and the draw over the whole row.
template <typename T>
__device__ void finish_row(const Row<T>& row, const Settings& s, float u, const Scale& sc, Shared& sm,
                           const Result& out) {
    const Weigh& w = out.w;
    uint64_t cut = 1;  // every unmasked item
    if (s.k) {
        clear(sm.hist, BINS);
        row.each([&](float z, uint32_t) { add(&sm.hist[sc.bin(z)], 1); });
        cut = cut_by_bins(row, sc, sm, uint64_t(s.k), [](float) { return uint64_t(1); });
    }
    if (s.p < 1.0f) {
        clear(sm.hist, BINS);
        uint64_t own = 0;
        row.each([&](float z, uint32_t i) {
            if (item_of(z, i) < cut) return;
            const uint64_t m = w.mass(z);
            own += m;
            if (m) add(&sm.hist[sc.bin(z)], m);
        });
        const uint64_t total = block_sum(own, sm);
        // (a mass of top_k's cut that lies past top_p's is not reached)
        const uint64_t c = cut_by_bins(row, sc, sm, share_of(s.p, total), [&](float z) { return w.mass(z); });
        cut = c > cut ? c : cut;
    }
    auto kept = [&](float z, uint32_t i) -> uint64_t {
        if (item_of(z, i) < cut) return 0;
        const double x = w(z);
        return x >= s.least ? Weigh::fixed(x) : 0;
    };
    __syncthreads();
    row.sums(sm.item, kept);
    const int ns = row.segments();
    uint64_t own = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < ns; i += NT) own += sm.item[i];
    const uint64_t total = block_sum(own, sm), target = goal(u, total);
    pick<false>(sm.item, ns, target, sm);
    draw_in(row.p, row.n, int64_t(sm.bin) * SEG, SEG, target - sm.before, total, out, kept);
}

__device__ inline void nothing_left(const Result& out) {
    *out.token = -1;
    if (out.logprob) *out.logprob = -INFINITY;
}

// Rows of at most SHORT logits: one workgroup a row.
template <typename T>
__global__ __launch_bounds__(NT) void sample_short(SampleArgs a) {
    __shared__ Shared sm;
    __shared__ float groups[SHORT / GROUP];
    const int64_t r = blockIdx.x;
    const int tid = int(threadIdx.x);
    const Row<T> row(static_cast<const T*>(a.logits) + r * a.ld, a.vocab);
    const Settings s = settings_of(a, r);
    const float u = a.u[r];
    if (tid == 0) sm.kmax = 0, sm.kfirst = 0xffffffffu;
    float zmax = -INFINITY;
    uint32_t first = 0xffffffffu;
    row.turns([&](const float* z, int64_t i) {
        float m = fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3]));
        if (m > zmax) {
            zmax = m;
            first = uint32_t(i) + (z[0] == m ? 0 : z[1] == m ? 1 : z[2] == m ? 2 : 3);
        }
        m = fmaxf(m, dpp_f32<0xb1>(m));  // (four lanes of a quad: a group)
        m = fmaxf(m, dpp_f32<0x4e>(m));
        if (tid % 4 == 0 && i < a.vocab) groups[i / GROUP] = m;
    });
    const float wmax = wave_max(zmax);
    __syncthreads();
    if (tid % WAVE == 0) atomicMax(&sm.kmax, key_of(wmax));
    __syncthreads();
    const uint32_t kmax = sm.kmax;
    const float top = value_of(kmax);
    const Result out{a.tokens + r, a.logprob ? a.logprob + r : nullptr, {double(top), s.inv_t}};
    if (kmax == 0) {
        if (tid == 0) nothing_left(out);
        return;
    }
    if (s.greedy) {
        if (zmax == top) atomicMin(&sm.kfirst, first);
        __syncthreads();
        if (tid == 0) out.certain(sm.kfirst);
        return;
    }
    const Scale sc(top, s.t);
    if (s.k || s.p < 1.0f || s.least > 0.0) {
        uint64_t total = 0;
        if (s.need_sum()) {
            uint64_t own = 0;
            row.each([&](float z, uint32_t) { own += out.w.mass(z); });
            total = block_sum(own, sm);
        }
        const int n = make_list(s, sc, sm, total, row, groups, out.w);
        if (n >= 0) {
            finish_list(n, s, u, total, sm, out);
            return;
        }
    }
    finish_row(row, s, u, sc, sm, out);
}

// What sample_stats leaves of a long row's 2,048 logits.
struct Chunk {
    float max;
    uint32_t first;  // index of the first maximum
    double sum;      // of exp((z - max) / T), where need_sum()
};

template <typename T, int VEC>
__global__ __launch_bounds__(256) void sample_stats(SampleArgs a, Chunk* chunks, float* groups, int64_t nchunk) {
    constexpr int L = CHUNK / WAVE / VEC, G = GROUP / VEC;  // loads of a lane; lanes of a group
    const int lane = int(threadIdx.x) % WAVE;
    const int64_t id = int64_t(blockIdx.x) * 4 + int(threadIdx.x) / WAVE;
    if (id >= a.rows * nchunk) return;
    const int64_t r = id / nchunk, c = id - r * nchunk;
    const T* p = static_cast<const T*>(a.logits) + r * a.ld;
    float z[L][VEC];
#pragma unroll
    for (int j = 0; j < L; ++j) {
        const int64_t i = c * CHUNK + (j * WAVE + lane) * VEC;
        if (i + VEC <= a.vocab) {
            typedef T vec __attribute__((ext_vector_type(VEC)));
            const vec v = *reinterpret_cast<const vec*>(p + i);
#pragma unroll
            for (int e = 0; e < VEC; ++e) z[j][e] = float(v[e]);
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) z[j][e] = i + e < a.vocab ? float(p[i + e]) : -INFINITY;
        }
    }
    const Settings s = settings_of(a, r);
    float top = -INFINITY;
    float* gr = groups + r * nchunk * (CHUNK / GROUP) + c * (CHUNK / GROUP);
#pragma unroll
    for (int j = 0; j < L; ++j) {
        float m = -INFINITY;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            z[j][e] = clean(z[j][e]);
            m = fmaxf(m, z[j][e]);
        }
        top = fmaxf(top, m);
#pragma unroll
        for (int o = 1; o < G; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, WAVE));
        if (lane % G == 0) gr[(j * WAVE + lane) / G] = m;
    }
    top = wave_max(top);
    uint32_t first = 0xffffffffu;
#pragma unroll
    for (int j = L - 1; j >= 0; --j)
#pragma unroll
        for (int e = VEC - 1; e >= 0; --e)
            if (z[j][e] == top) first = uint32_t(c * CHUNK + (j * WAVE + lane) * VEC + e);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const uint32_t x = __shfl_xor(first, o, WAVE);
        first = x < first ? x : first;
    }
    double sum = 0.0;
    if (s.need_sum() && top > -INFINITY) {
        const Weigh w{double(top), s.inv_t};
#pragma unroll
        for (int j = 0; j < L; ++j)
#pragma unroll
            for (int e = 0; e < VEC; ++e) sum += w(z[j][e]);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, WAVE);
    }
    if (lane == 0) chunks[id] = Chunk{top, first, sum};
}

// Long rows whose kept tokens do not fit a list, between the kernels.
struct Pending {
    uint64_t cut;       // the first item that goes
    uint32_t kmax;
    uint32_t step;      // 0: done; 1: the cut is to be found; 2: the draw
    uint32_t arrived[2];
};
struct Workspace {
    Chunk* chunks;      // [rows][nchunk]
    float* groups;      // [rows][nchunk * CHUNK / GROUP]
    Pending* pending;   // [rows]
    uint64_t* hist;     // [rows][BINS]
    uint64_t* segs;     // [rows][nchunk * CHUNK / SEG]
    int64_t nchunk;
    Workspace from(int64_t r) const {
        Workspace w = *this;
        w.chunks += r * nchunk, w.groups += r * nchunk * (CHUNK / GROUP), w.pending += r;
        w.hist += r * BINS, w.segs += r * nchunk * (CHUNK / SEG);
        return w;
    }
};

constexpr int PART = 16 * NT;  // logits of a workgroup of the wide kernels

template <typename T>
__global__ __launch_bounds__(NT) void sample_long(SampleArgs a, Workspace ws) {
    __shared__ Shared sm;
    const int64_t r = blockIdx.x, nchunk = ws.nchunk;
    const int tid = int(threadIdx.x);
    const Settings s = settings_of(a, r);
    const float u = a.u[r];
    const Chunk* chunks = ws.chunks + r * nchunk;
    const float* groups = ws.groups + r * nchunk * (CHUNK / GROUP);
    const Row<T> row(static_cast<const T*>(a.logits) + r * a.ld, a.vocab);
    if (tid == 0) sm.kmax = 0, sm.kfirst = 0xffffffffu, ws.pending[r].step = 0;
    __syncthreads();
    const Chunk mine = tid < nchunk ? chunks[tid] : Chunk{-INFINITY, 0xffffffffu, 0.0};  // (nchunk <= NT)
    const float wmax = wave_max(mine.max);
    if (tid % WAVE == 0) atomicMax(&sm.kmax, key_of(wmax));
    __syncthreads();
    const uint32_t kmax = sm.kmax;
    const float top = value_of(kmax);
    Result out{a.tokens + r, a.logprob ? a.logprob + r : nullptr, {double(top), s.inv_t}};
    if (kmax == 0) {
        if (tid == 0) nothing_left(out);
        return;
    }
    if (s.greedy) {
        if (mine.max == top) atomicMin(&sm.kfirst, mine.first);
        __syncthreads();
        if (tid == 0) out.certain(sm.kfirst);
        return;
    }
    uint64_t own = 0, total = 0;
    if (s.need_sum()) {
        // (a chunk has a mass where one of its logits has)
        const double x = out.w(mine.max);
        if (Weigh::fixed(x)) own = uint64_t(rint(mine.sum * x * ONE));
        total = block_sum(own, sm);
    }
    if (s.k == 0 && s.p >= 1.0f && s.least == 0.0) {
        sm.hist[tid] = own;
        const uint64_t target = goal(u, total);
        pick<false>(sm.hist, NT, target, sm);
        const int64_t c = sm.bin;
        const uint64_t left = target - sm.before;
        // the chunk's segments, then the segment
        const Row<T> part(row.p + c * CHUNK, a.vocab - c * CHUNK < CHUNK ? a.vocab - c * CHUNK : CHUNK);
        auto mass = [&](float z, uint32_t) { return out.w.mass(z); };
        __syncthreads();
        part.sums(sm.item, mass);
        pick<false>(sm.item, part.segments(), left, sm);
        // (the chunk's sum and its logits' masses differ by their rounding:
        // past the end is the last logit with a mass)
        int seg = int(sm.bin);
        uint64_t target2 = left > sm.before ? left - sm.before : 1;
        if (sm.total < left) {
            while (seg > 0 && sm.item[seg] == 0) --seg;
            target2 = sm.item[seg];
        }
        draw_in(row.p, a.vocab, c * CHUNK + int64_t(seg) * SEG, SEG, target2, total, out, mass);
        return;
    }
    const Scale sc(top, s.t);
    const int n = make_list(s, sc, sm, total, row, groups, out.w);
    if (n >= 0) {
        finish_list(n, s, u, total, sm, out);
        return;
    }
    if (s.k) {
        finish_row(row, s, u, sc, sm, out);
        return;
    }
    for (int i = tid; i < BINS; i += NT) ws.hist[r * BINS + i] = 0;
    if (tid == 0) ws.pending[r] = Pending{1, kmax, s.p < 1.0f ? 1u : 2u, {0, 0}};
}

// Whether this workgroup is the last of its row's to arrive; what the others
// wrote before is then visible to it.  (One thread fences for all, ordered
// with them by the barriers: a fence writes back and invalidates the L2, and
// one by every wave took 300 us of a 16.8 million logits' pass.)
__device__ inline bool last_of(uint32_t* arrived, Shared& sm) {
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        sm.count = int(atomicAdd(arrived, 1u));
        __threadfence();
    }
    __syncthreads();
    const bool last = sm.count == int(gridDim.x) - 1;
    __syncthreads();
    return last;
}
__device__ inline uint64_t load_shared(const uint64_t* p) {  // written by other workgroups of this launch
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The logits of this workgroup's part of a row.
__device__ inline int64_t part_size(int64_t n) {
    const int64_t left = n - int64_t(blockIdx.x) * PART;
    return left < PART ? left : PART;
}

// The masses of pending rows by bins; the last workgroup of a row finds
// top_p's cut.
template <typename T>
__global__ __launch_bounds__(NT) void sample_bins(SampleArgs a, Workspace ws) {
    const int64_t r = blockIdx.y;
    Pending& pd = ws.pending[r];
    if (pd.step != 1) return;
    __shared__ Shared sm;
    const int tid = int(threadIdx.x);
    const Settings s = settings_of(a, r);
    const Row<T> row(static_cast<const T*>(a.logits) + r * a.ld, a.vocab);
    const float top = value_of(pd.kmax);
    const Weigh w{double(top), s.inv_t};
    const Scale sc(top, s.t);
    clear(sm.hist, BINS);
    const Row<T> part(row.p + int64_t(blockIdx.x) * PART, part_size(row.n));
    part.each([&](float z, uint32_t) {
        const uint64_t m = w.mass(z);
        if (m) add(&sm.hist[sc.bin(z)], m);
    });
    __syncthreads();
    uint64_t* hist = ws.hist + r * BINS;
    for (int i = tid; i < BINS; i += NT)
        if (sm.hist[i]) add(hist + i, sm.hist[i]);
    if (!last_of(&pd.arrived[0], sm)) return;
    uint64_t own = 0;
    for (int i = tid; i < BINS; i += NT) {
        sm.hist[i] = load_shared(hist + i);
        own += sm.hist[i];
    }
    const uint64_t total = block_sum(own, sm);
    const uint64_t cut = cut_by_bins(row, sc, sm, share_of(s.p, total), [&](float z) { return w.mass(z); });
    if (tid == 0) pd.cut = cut, pd.step = 2;
}

// The kept masses of pending rows by segments; the last workgroup of a row
// draws.
template <typename T>
__global__ __launch_bounds__(NT) void sample_draw(SampleArgs a, Workspace ws) {
    const int64_t r = blockIdx.y;
    Pending& pd = ws.pending[r];
    if (pd.step != 2) return;
    __shared__ Shared sm;
    const int tid = int(threadIdx.x);
    const Settings s = settings_of(a, r);
    const T* p = static_cast<const T*>(a.logits) + r * a.ld;
    const Result out{a.tokens + r, a.logprob ? a.logprob + r : nullptr, {double(value_of(pd.kmax)), s.inv_t}};
    const uint64_t cut = pd.cut;
    auto kept = [&](float z, uint32_t i) -> uint64_t {
        if (item_of(z, i) < cut) return 0;
        const double x = out.w(z);
        return x >= s.least ? Weigh::fixed(x) : 0;
    };
    const int64_t first = int64_t(blockIdx.x) * PART, ns = ws.nchunk * (CHUNK / SEG);
    uint64_t* segs = ws.segs + r * ns;
    const Row<T> part(p + first, part_size(a.vocab));
    // (the segments of a part end with the row, the row's with its chunks)
    part.sums(sm.item, [&](float z, uint32_t i) { return kept(z, uint32_t(first) + i); });
    __syncthreads();
    for (int i = tid; i < PART / SEG && first / SEG + i < ns; i += NT)
        __hip_atomic_store(segs + first / SEG + i, i < part.segments() ? sm.item[i] : 0, __ATOMIC_RELAXED,
                           __HIP_MEMORY_SCOPE_AGENT);
    if (!last_of(&pd.arrived[1], sm)) return;
    uint64_t own = 0;
    for (int i = tid; i < ns; i += NT) {
        sm.item[i] = load_shared(segs + i);
        own += sm.item[i];
    }
    const uint64_t total = block_sum(own, sm), target = goal(a.u[r], total);
    pick<false>(sm.item, int(ns), target, sm);
    draw_in(p, a.vocab, int64_t(sm.bin) * SEG, SEG, target - sm.before, total, out, kept);
}

void check(const SampleArgs& a) {
    if (a.dtype != ELEM_F32 && a.dtype != ELEM_F16 && a.dtype != ELEM_BF16)
        fail(E_INVALID, "sample: logits must be f32, f16 or bf16");
    if (a.rows <= 0 || a.rows > (1 << 24)) fail(E_INVALID, "sample: rows must be 1 to 2^24");
    if (a.vocab <= 0 || a.vocab > (1 << IDX_BITS)) fail(E_INVALID, "sample: vocab must be 1 to 2^20");
}

template <typename T>
SampleArgs rows_from(SampleArgs a, int64_t r) {
    a.logits = static_cast<const T*>(a.logits) + r * a.ld;
    a.u += r, a.tokens += r;
    if (a.logprob) a.logprob += r;
    if (a.temperature) a.temperature += r;
    if (a.top_k) a.top_k += r;
    if (a.top_p) a.top_p += r;
    if (a.min_p) a.min_p += r;
    return a;
}

int64_t chunks_of(int64_t vocab) { return (vocab + CHUNK - 1) / CHUNK; }

template <typename T>
void launch(hipStream_t s, const SampleArgs& a, void* workspace) {
    const dim3 grid{unsigned(a.rows)}, block{NT};
    if (a.vocab <= SHORT) {
        sample_short<T><<<grid, block, 0, s>>>(a);
    } else {
        const int64_t nchunk = chunks_of(a.vocab);
        Workspace ws;
        ws.nchunk = nchunk;
        ws.chunks = static_cast<Chunk*>(workspace);
        ws.hist = reinterpret_cast<uint64_t*>(ws.chunks + a.rows * nchunk);
        ws.segs = ws.hist + a.rows * BINS;
        ws.pending = reinterpret_cast<Pending*>(ws.segs + a.rows * nchunk * (CHUNK / SEG));
        ws.groups = reinterpret_cast<float*>(ws.pending + a.rows);
        const dim3 wide{unsigned((a.rows * nchunk + 3) / 4)};
        constexpr int VEC = 16 / int(sizeof(T));
        if (reinterpret_cast<uintptr_t>(a.logits) % 16 == 0 && a.ld % VEC == 0)
            sample_stats<T, VEC><<<wide, dim3(256), 0, s>>>(a, ws.chunks, ws.groups, nchunk);
        else
            sample_stats<T, 1><<<wide, dim3(256), 0, s>>>(a, ws.chunks, ws.groups, nchunk);
        OMG_HIP(hipGetLastError());
        sample_long<T><<<grid, block, 0, s>>>(a, ws);
        if (a.top_p || a.min_p) {
            OMG_HIP(hipGetLastError());
            for (int64_t r = 0; r < a.rows; r += 65535) {  // (a grid's second size)
                const dim3 parts{unsigned((a.vocab + PART - 1) / PART), unsigned(std::min<int64_t>(65535, a.rows - r))};
                const SampleArgs b = rows_from<T>(a, r);
                const Workspace wr = ws.from(r);
                if (a.top_p) sample_bins<T><<<parts, block, 0, s>>>(b, wr);
                OMG_HIP(hipGetLastError());
                sample_draw<T><<<parts, block, 0, s>>>(b, wr);
                OMG_HIP(hipGetLastError());
            }
        }
    }
    OMG_HIP(hipGetLastError());
}

}  // namespace

int64_t sample_workspace(int64_t rows, int64_t vocab) {
    SampleArgs a{};
    a.rows = rows, a.vocab = vocab;
    check(a);
    static_assert(sizeof(Pending) % 8 == 0 && sizeof(Chunk) % 16 == 0, "the workspace's arrays are aligned");
    return vocab <= SHORT ? 0
                          : rows * (chunks_of(vocab) * int64_t(sizeof(Chunk) + CHUNK / SEG * 8 + CHUNK / GROUP * 4) +
                                    BINS * 8 + int64_t(sizeof(Pending)));
}

void launch_sample(hipStream_t s, const SampleArgs& a, void* workspace, size_t bytes) {
    const int64_t need = sample_workspace(a.rows, a.vocab);
    check(a);
    if (a.ld < a.vocab) fail(E_INVALID, "sample: ld must hold the vocabulary");
    if (!a.logits || !a.u || !a.tokens) fail(E_INVALID, "sample: null logits, u or tokens");
    if (reinterpret_cast<uintptr_t>(a.logits) % (a.dtype == ELEM_F32 ? 4 : 2))
        fail(E_INVALID, "sample: logits must be aligned to their type");
    if (int64_t(bytes) < need) fail(E_CAPACITY, "sample: the workspace needs " + std::to_string(need) + " bytes");
    if (need && (!workspace || !aligned16(workspace)))
        fail(E_INVALID, "sample: the workspace must be 16-byte aligned");
    if (a.dtype == ELEM_F32)
        launch<float>(s, a, workspace);
    else if (a.dtype == ELEM_F16)
        launch<half_t>(s, a, workspace);
    else
        launch<bf16_t>(s, a, workspace);
}

}  // namespace omg
