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
// once by the whole chip (sample_stats: per 1,024 logits the maximum, its
// index and, where the row's filters need it, the sum of exp; per 16 the
// maximum), then one workgroup a row looks at these (sample_long).  Both look
// for a threshold that few logits pass but all that can be kept do, from the
// maxima of groups of 16: the k-th largest of these maxima has k logits at or
// above it; min_p's threshold is its own; for top_p alone a guess is taken
// and proved by the mass above it.  The logits above it are gathered into a
// list in LDS, where the exact cuts and the drawn token are found by
// comparing all pairs (up to 256) or by histograms over the items' digits.
// Where the kept tokens do not fit the list, the row's masses are summed by
// bins of their distance from the maximum, which leaves one bin's logits to
// order exactly, and the kept masses by segments in index order: by one
// workgroup a row (finish_row: short rows, and top_k of long ones), or by the
// whole chip (sample_bins, sample_draw: top_p and min_p of long rows).
//
// What bounds the kernels of one workgroup a row is its CU: 64 lanes a cycle
// (150 lane instructions a nanosecond) and a microsecond for every trip to
// memory that the next step waits for.  So passes over a row compare raw
// logits with a threshold and take keys, bins and masses of the few that
// pass, and their loops are rolled: a row of 25,000 held in registers, 32 a
// thread, took 14.5 us for its maximum and 14 for a pass of exp, waiting for
// instructions; this form takes 5.
//
// Measured: one row of 25,000 15.4 us (f32; top_k 40, top_p 0.95: seven steps
// that wait for one another); 208 of them, each with its own filters, 52 us
// (the rows whose kept tokens fit no list); 64 rows of 262,144 (bf16, top_p)
// 104 us: stats 24 (37 vector instructions a logit, most of them exp's),
// long 20, bins 26, draw 39 (the last rows' cuts, one workgroup each); 256
// rows of 128,257 (f32, mixed filters) 111 us, of which stats 33 (3.9 TB/s).
#include <algorithm>
#include <string>

#include "common.h"
#include "kern_common.h"
#include "paged.h"

namespace omg {

namespace {

constexpr int NT = 1024;          // threads of a row's workgroup
constexpr int NWAVE = NT / WAVE;
constexpr int CHUNK = 1024;       // logits of a wave of sample_stats
constexpr int GROUP = 16;         // logits of a group maximum
constexpr int SHORT = 32 * NT;    // logits of a row that one workgroup takes alone
constexpr int CAP = 8192;         // items of the list
constexpr int BINS = 2048;
constexpr int PAIRS = NT / 4;     // items compared pair by pair: four threads each
constexpr int SEG = 256;          // consecutive logits a wave takes at once
constexpr int PART = 16 * NT;     // logits of a workgroup of the wide kernels
constexpr int EDGE = 2048;        // logits of one bin that they set apart
constexpr int IDX_BITS = 20;      // vocab <= 2^20
constexpr uint32_t IDX_MASK = (1u << IDX_BITS) - 1;
constexpr double ONE = 4398046511104.0;  // 2^42
constexpr float LOWEST = -3.4028235e38f;

// Order-preserving bits of a logit that is not masked (above -infinity); -0
// is the 0 it equals.
__device__ inline uint32_t key_of(float z) {
    const uint32_t u = __builtin_bit_cast(uint32_t, z + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ inline float value_of(uint32_t k) {
    return __builtin_bit_cast(float, k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
// An item: larger comes first.
__device__ inline uint64_t item_of(float z, int i) { return uint64_t(key_of(z)) << IDX_BITS | (IDX_MASK - uint32_t(i)); }
__device__ inline float item_value(uint64_t it) { return value_of(uint32_t(it >> IDX_BITS)); }
__device__ inline int item_index(uint64_t it) { return int(IDX_MASK - (uint32_t(it) & IDX_MASK)); }

// The items from the first on to an item, as logits compare: larger ones, and
// its equals up to its index.  Without one: all that are not masked.
struct Cut {
    float z = -INFINITY;
    int i = 0;
    __device__ bool keeps(float x, int at) const { return x > z || (x == z && at <= i && z > -INFINITY); }
    static __device__ Cut at(uint64_t item) {
        Cut c;
        if (uint32_t(item >> IDX_BITS) > 0x007fffffu) c.z = item_value(item), c.i = item_index(item);  // (-infinity's key)
        return c;
    }
};

// exp((z - max) / T): 1 at the maximum, whatever it is, nothing where z is
// masked.  With t = (z - max) log2(e) / T = n + f, |f| <= 1/2: the series of
// 2^f = exp(f ln 2) to the 11th power (its rest is below 2^-46), its exponent
// raised by n.
struct Weigh {
    double max, per;  // log2(e) / T
    bool infinite;
    __device__ Weigh(float m, double inv_t)
        : max(double(m)), per(inv_t * 1.4426950408889634), infinite(m == INFINITY) {}
    __device__ double operator()(float z) const {
        if (infinite) return z == INFINITY ? 1.0 : 0.0;
        constexpr double WHOLE = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to a whole number
        // (NaN, and what is far below every mass, to 2^-1000)
        const double t = fmax((double(z) - max) * per, -1000.0);
        const double shifted = t + WHOLE, f = t - (shifted - WHOLE);
        constexpr double L = 0.69314718055994531;
        constexpr double c2 = L * L / 2, c3 = c2 * L / 3, c4 = c3 * L / 4, c5 = c4 * L / 5, c6 = c5 * L / 6,
                         c7 = c6 * L / 7, c8 = c7 * L / 8, c9 = c8 * L / 9, c10 = c9 * L / 10, c11 = c10 * L / 11;
        double p = c11;
        step(p, f, c10), step(p, f, c9), step(p, f, c8), step(p, f, c7), step(p, f, c6), step(p, f, c5);
        step(p, f, c4), step(p, f, c3), step(p, f, c2), step(p, f, L), step(p, f, 1.0);
        const uint64_t b = __builtin_bit_cast(uint64_t, p);
        const uint32_t n = uint32_t(__builtin_bit_cast(uint64_t, shifted));  // (its low bits: n)
        return __builtin_bit_cast(double, uint64_t(uint32_t(b >> 32) + (n << 20)) << 32 | uint32_t(b));
    }
    // p = p f + c, c in scalar registers (the compiler's form, which adds onto
    // its third operand, first moves each c into vector registers: 22 of 59
    // instructions a logit).
    static __device__ void step(double& p, double f, double c) {
        asm("v_fma_f64 %0, %0, %1, %2" : "+v"(p) : "v"(f), "s"(c));
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

// Sums over the wave by DPP (a shuffle goes through LDS, a hundred cycles a
// step): lanes without a source add 0.
template <int CTRL, int ROWS>
__device__ inline uint64_t dpp_u64(uint64_t v) {
    const uint32_t lo = uint32_t(__builtin_amdgcn_update_dpp(0, int(uint32_t(v)), CTRL, ROWS, 0xf, true));
    const uint32_t hi = uint32_t(__builtin_amdgcn_update_dpp(0, int(uint32_t(v >> 32)), CTRL, ROWS, 0xf, true));
    return uint64_t(hi) << 32 | lo;
}
__device__ inline uint64_t row_scan_u64(uint64_t v) {  // inclusive, in each 16 lanes
    v += dpp_u64<0x111, 0xf>(v);  // row_shr 1, 2, 4, 8
    v += dpp_u64<0x112, 0xf>(v);
    v += dpp_u64<0x114, 0xf>(v);
    v += dpp_u64<0x118, 0xf>(v);
    return v;
}
__device__ inline uint64_t wave_scan_u64(uint64_t v) {  // inclusive
    v = row_scan_u64(v);
    v += dpp_u64<0x142, 0xa>(v);  // row_bcast 15: into rows 1 and 3
    v += dpp_u64<0x143, 0xc>(v);  // row_bcast 31: into rows 2 and 3
    return v;
}
__device__ inline uint64_t quad_sum_u64(uint64_t v) {  // over four lanes, in each
    v += dpp_u64<0xb1, 0xf>(v);
    v += dpp_u64<0x4e, 0xf>(v);
    return v;
}
__device__ inline uint64_t lane_u64(uint64_t v, int lane) {
    const uint32_t lo = uint32_t(__builtin_amdgcn_readlane(int(uint32_t(v)), lane));
    const uint32_t hi = uint32_t(__builtin_amdgcn_readlane(int(uint32_t(v >> 32)), lane));
    return uint64_t(hi) << 32 | lo;
}

struct Common {
    uint64_t part[NWAVE];
    uint64_t before, in_bin, total, found;
    uint32_t bin, kmax, kfirst, count;
    int row_n;  // the row's logits (as an argument 27 more scalars spilled: one row of 25,000 15.4 -> 17.2 us)
};
// Lists of logits that pass a threshold, one a wave.
struct Passed {
    float z[NWAVE][5 * WAVE];
    int at[NWAVE][5 * WAVE];
};
struct Shared : Common {
    uint64_t item[CAP];   // the list; without one, the masses of the row's segments
    union {
        uint64_t mass[CAP];   // kept masses; before, the numbers of the groups to read
        Passed list;
    };
    uint64_t hist[BINS];
    uint64_t edge[PAIRS]; // items of one bin
};
struct BinsShared : Common {
    uint64_t hist[BINS];
    Passed list;
};
struct DrawShared : Common {
    union {
        struct {
            uint64_t item[(1 << IDX_BITS) / SEG];  // the masses of the row's segments
            uint64_t hist[BINS];
        };
        Passed list;
    };
    uint64_t seg[PART / SEG];  // of this part's
    uint64_t edge[EDGE];
};
__device__ inline int wave_id() { return __builtin_amdgcn_readfirstlane(int(threadIdx.x) / WAVE); }

// Sum of v over the workgroup, in every thread.
__device__ inline uint64_t block_sum(uint64_t v, Common& sm) {
    const int lane = int(threadIdx.x) % WAVE;
    v = wave_scan_u64(v);
    __syncthreads();
    if (lane == WAVE - 1) sm.part[wave_id()] = v;
    __syncthreads();
    return lane_u64(row_scan_u64(sm.part[lane % NWAVE]), NWAVE - 1);
}

// The bin at which the running sum over h[0 .. n), in ascending or (DOWN)
// descending order, first reaches `target`; the last one in order if it
// never does.  Sets sm.bin, sm.before (the sum before it), sm.in_bin and
// sm.total.  n up to 4 NT.
template <bool DOWN>
__device__ inline void pick(const uint64_t* h, int n, uint64_t target, Common& sm) {
    const int tid = int(threadIdx.x), lane = tid % WAVE, wave = wave_id();
    const int per = (n + NT - 1) / NT;
    __syncthreads();
    uint64_t x[4], own = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int j = tid * per + i;
        x[i] = i < per && j < n ? h[DOWN ? n - 1 - j : j] : 0;
        own += x[i];
    }
    const uint64_t scan = wave_scan_u64(own);
    if (lane == WAVE - 1) sm.part[wave] = scan;
    __syncthreads();
    const uint64_t waves = row_scan_u64(sm.part[lane % NWAVE]);
    const uint64_t total = lane_u64(waves, NWAVE - 1);
    uint64_t run = (wave ? lane_u64(waves, wave - 1) : 0) + scan - own;
    const bool never = total < target;
    if (tid == 0) sm.total = total;
    if (never ? tid == (n - 1) / per : run < target && run + own >= target) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int j = tid * per + i;
            if (i < per && (never ? j == n - 1 : run < target && run + x[i] >= target)) {
                sm.bin = uint32_t(DOWN ? n - 1 - j : j);
                sm.before = run;
                sm.in_bin = x[i];
            }
            run += x[i];
        }
    }
    __syncthreads();
}

// (h's last readers are past a barrier)
__device__ inline void clear(uint64_t* h, int n) {
    for (int i = threadIdx.x; i < n; i += NT) h[i] = 0;
    __syncthreads();
}
__device__ inline void add(uint64_t* h, uint64_t v) {
    atomicAdd(reinterpret_cast<unsigned long long*>(h), static_cast<unsigned long long>(v));
}

// A place in a list for each of the lane's `own` entries, by one atomic of
// the wave.
__device__ inline int places(uint32_t* count, int own) {
    int scan = own;
    scan += __builtin_amdgcn_update_dpp(0, scan, 0x111, 0xf, 0xf, true);
    scan += __builtin_amdgcn_update_dpp(0, scan, 0x112, 0xf, 0xf, true);
    scan += __builtin_amdgcn_update_dpp(0, scan, 0x114, 0xf, 0xf, true);
    scan += __builtin_amdgcn_update_dpp(0, scan, 0x118, 0xf, 0xf, true);
    scan += __builtin_amdgcn_update_dpp(0, scan, 0x142, 0xa, 0xf, true);
    scan += __builtin_amdgcn_update_dpp(0, scan, 0x143, 0xc, 0xf, true);
    const int all = __builtin_amdgcn_readlane(scan, WAVE - 1);
    uint32_t at = 0;
    if (all && threadIdx.x % WAVE == 0) at = atomicAdd(count, uint32_t(all));
    return __builtin_amdgcn_readfirstlane(int(at)) + scan - own;
}


// Bins of the distance from the row's maximum, T / 64 or 1/32 wide, whichever
// is narrower.
struct Scale {
    float max, per;  // bins per unit of z
    bool whole;      // what lies in the last bin has no mass
    __device__ Scale(float m, float t) : max(m) {
        const float f = 64.0f / t;
        per = f > 32.0f ? (f < 1e30f ? f : 1e30f) : 32.0f;
        whole = float(BINS - 1) > 30.5f * t * per;  // e^-29.9 < 2^-43
    }
    __device__ int bin(float z) const {
        const float x = (max - z) * per;
        return x < float(BINS - 1) ? int(x) : BINS - 1;  // (NaN, infinity - infinity: the last)
    }
    // The bins that top_p's cut can lie in, of the n logits that p is a share
    // of, whose mass is at least `mass` of the largest's: those below the last
    // one returned weigh less than (1 - p) mass / (2 n) each, together less
    // than half of what top_p leaves.  The other half is for the masses'
    // rounding, up to 2^-42 a logit in the sums compared: all bins where that
    // is more.
    __device__ int reach(float p, float mass, int n, float t) const {
        const float leaves = (1.0f - p) * mass;
        if (!(leaves > 5e-13f * float(n))) return BINS - 1;  // (2^-41)
        const float nats = logf(2.0f * float(n) / leaves);
        const float x = nats * t * per + 2.0f;
        return x < float(BINS - 1) && max < INFINITY ? int(x) : BINS - 1;  // (infinities lie in the last)
    }
    // The bins that min_p can keep, and one to spare.
    __device__ int reach_min(double least, float t) const {
        const float far = float(-log(least) * double(t)) * per + 1.0f;
        return far < float(BINS - 2) ? int(far) + 1 : BINS - 1;
    }
    // A logit below all that lie in bins 0 .. last, however the bins rounded.
    __device__ float under(int last) const {
        const float x = max - float(last + 1) / per * 1.00001f;
        return x - fabsf(x) * 1e-6f - 1e-37f;
    }
    // The same, finite; the lowest logit where the last bin is among them.
    __device__ float low(int last) const { return last < BINS - 1 ? fmaxf(under(last), LOWEST) : LOWEST; }
};

// A row of logits: raw, masked ones as they stand (NaN, -infinity).
template <typename T>
struct Row {
    const T* p;
    int n;
    bool wide;  // four elements at once are aligned
    typedef T vec __attribute__((ext_vector_type(4)));
    __device__ Row(const T* row, int64_t vocab)
        : p(row), n(int(vocab)), wide(reinterpret_cast<uintptr_t>(row) % (4 * sizeof(T)) == 0 && vocab >= 4) {}
    // The four logits from i (a multiple of 4) on, -infinity behind the row,
    // in two steps, so that a caller's loads can be under way together.
    __device__ vec load(int i) const {
        if (wide) return *reinterpret_cast<const vec*>(p + (i + 4 <= n ? i : 0));
        vec v;
#pragma unroll
        for (int c = 0; c < 4; ++c) v[c] = p[i + c < n ? i + c : 0];
        return v;
    }
    __device__ void four(vec v, int i, float* z) const {
#pragma unroll
        for (int c = 0; c < 4; ++c) z[c] = float(v[c]);
        if (i + 4 > n) {
#pragma unroll
            for (int c = 0; c < 4; ++c) z[c] = i + c < n ? float(p[i + c]) : -INFINITY;
        }
    }
    // f(z, i) for the four logits z of each of the thread's turns, the next
    // two turns' loads under way; every thread makes the same turns, a wave
    // takes SEG consecutive logits in each.
    template <typename F>
    __device__ void turns(F&& f) const {
        int i = int(threadIdx.x) * 4;
        vec v0 = load(i), v1 = load(i + NT * 4);
#pragma unroll 1
        for (int base = 0; base < n; base += NT * 8, i += NT * 8) {
            const vec w0 = load(i + NT * 8), w1 = load(i + NT * 12);
            float z[4];
            four(v0, i, z);
            f(z, i);
            four(v1, i + NT * 4, z);
            f(z, i + NT * 4);
            v0 = w0, v1 = w1;
        }
    }
    __device__ int segments() const { return (n + SEG - 1) / SEG; }
    // Sums of m(z, i) over the row's segments.
    template <typename F>
    __device__ void sums(uint64_t* out, F&& m) const {
        turns([&](const float* z, int i) {
            uint64_t v = 0;
#pragma unroll
            for (int c = 0; c < 4; ++c) v += m(z[c], i + c);
            v = wave_scan_u64(v);
            if (threadIdx.x % WAVE == WAVE - 1 && i - (WAVE - 1) * 4 < n) out[i / SEG] = v;
        });
    }
};

struct Result {
    int32_t* token;
    float* logprob;
    Weigh w;
    double inv_t;
    __device__ Result(const SampleArgs& a, int64_t r, float max, const Settings& s)
        : token(a.tokens + r), logprob(a.logprob ? a.logprob + r : nullptr), w(max, s.inv_t), inv_t(s.inv_t) {}
    __device__ void certain(int i) const {
        *token = i;
        if (logprob) *logprob = i < 0 ? -INFINITY : 0.0f;
    }
    __device__ void write(float z, int i, uint64_t total) const {
        *token = i;
        const double d = double(z) - w.max;
        if (logprob) *logprob = float((d < 0.0 ? d * inv_t : 0.0) - log(double(total) / ONE));
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
__device__ inline void draw_in(const Row<T>& row, int first, uint64_t target, uint64_t total, const Result& out, F&& m) {
    if (threadIdx.x >= WAVE) return;
    const int lane = int(threadIdx.x), i = first + lane * 4;
    float z[4];
    row.four(row.load(i), i, z);
    uint64_t v[4], own = 0;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        v[c] = m(z[c], i + c);
        own += v[c];
    }
    const uint64_t scan = wave_scan_u64(own);
    const uint64_t some = __ballot(own > 0), hit = __ballot(own > 0 && scan >= target);
    if (!some || lane != (hit ? __builtin_ctzll(hit) : 63 - __builtin_clzll(some))) return;
    uint64_t run = scan - own;
    float drawn = 0.0f;
    int at = -1;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const bool here = v[c] > 0 && (at < 0 || run < target);
        if (here) drawn = z[c], at = i + c;
        run += v[c];
    }
    out.write(drawn, at, total);
}

// The item at which the running share, over the items from the first on,
// first reaches `target` (>= 1); 0 if it never does, or an item below all
// that do.  items(f) calls f(z, i) for the thread's items; masses: an item's
// share is its mass, else one.
template <typename S, typename M>
__device__ uint64_t find_cut(S&& items, M& sm, uint64_t target, bool masses, const Weigh& w) {
    uint64_t prefix = 0, before = 0;
    int shift = 52;
#pragma unroll 1
    for (int level = 0; level < 5; ++level) {
        const int bits = level < 2 ? 11 : 10;
        shift -= bits;
        clear(sm.hist, 1 << bits);
        items([&](float z, int i) {
            const uint64_t it = item_of(z, i);
            if ((it >> (shift + bits)) != prefix) return;
            const uint64_t v = masses ? w.mass(z) : 1;
            if (v) add(&sm.hist[(it >> shift) & ((1u << bits) - 1)], v);
        });
        pick<true>(sm.hist, 1 << bits, target - before, sm);
        prefix = prefix << bits | sm.bin;
        before += sm.before;
        if (before + sm.in_bin <= target) break;  // the whole bin stays
    }
    return prefix << shift;
}

// The cut within one bin: room[0 .. n) are its items, `left` the share that
// is taken from them (reached among them).  Up to PAIRS items are compared
// pair by pair; of more, digits from the first that differs on leave as few.
template <typename M>
__device__ Cut cut_in_bin(const uint64_t* room, int n, M& sm, uint64_t left, bool masses, const Weigh& w) {
    const int tid = int(threadIdx.x);
    uint64_t* mass = sm.hist;
    const auto share = [&](uint64_t it) { return masses ? w.mass(item_value(it)) : 1; };
    __syncthreads();
    if (n > PAIRS) {
        if (tid == 0) sm.found = 0, sm.total = ~uint64_t(0);
        __syncthreads();
        uint64_t most = 0, least = ~uint64_t(0);
        for (int i = tid; i < n; i += NT) {
            const uint64_t it = room[i];
            most = most > it ? most : it, least = least < it ? least : it;
        }
        if (most) {
            atomicMax(reinterpret_cast<unsigned long long*>(&sm.found), static_cast<unsigned long long>(most));
            atomicMin(reinterpret_cast<unsigned long long*>(&sm.total), static_cast<unsigned long long>(least));
        }
        __syncthreads();
        int shift = 64 - __builtin_clzll(sm.found ^ sm.total);  // (items differ)
        uint64_t prefix = sm.found >> shift;
        uint64_t* few = sm.hist + BINS / 2;
        int count;
        do {
            const int bits = shift < 11 ? shift : 11;
            shift -= bits;
            clear(sm.hist, BINS);
            if (tid == 0) sm.count = 0;
            for (int i = tid; i < n; i += NT) {
                const uint64_t it = room[i], v = it >> (shift + bits) == prefix ? share(it) : 0;
                if (v) add(&sm.hist[it >> shift & ((1u << bits) - 1)], v);
            }
            pick<true>(sm.hist, 1 << bits, left, sm);
            prefix = prefix << bits | sm.bin;
            left -= sm.before;
            for (int i = tid; i < n; i += NT) {
                const uint64_t it = room[i];
                if (it >> shift != prefix) continue;
                const uint32_t at = atomicAdd(&sm.count, 1u);
                if (at < PAIRS) few[at] = it;
            }
            __syncthreads();
            count = int(sm.count);
        } while (count > PAIRS);
        room = few, n = count;
    }
    if (tid == 0) sm.found = 0;
    if (tid < n) mass[tid] = share(room[tid]);
    __syncthreads();
    const int e = tid / 4, lane4 = tid % 4;
    if (e < n) {
        const uint64_t mine = room[e], own = mass[e];
        uint64_t run = 0;
#pragma unroll 4
        for (int j = lane4; j < n; j += 4) run += room[j] >= mine ? mass[j] : 0;
        run = quad_sum_u64(run);
        if (lane4 == 0 && own && run >= left && run - own < left) sm.found = mine;
    }
    __syncthreads();
    return Cut::at(sm.found);
}

// The cut at which the running share reaches `target`, the shares' sums by
// bins in sm.hist: the items of the bin where it does are collected, in
// room[0 .. most); past the room the digits decide over all items.
template <typename S>
__device__ Cut cut_by_bins(S&& items, const Scale& sc, Shared& sm, uint64_t* room, int most, uint64_t target,
                           bool masses, const Weigh& w) {
    pick<false>(sm.hist, BINS, target, sm);
    const int bin = int(sm.bin);
    const uint64_t left = target - sm.before;
    if (sm.total < target) return Cut();
    __syncthreads();
    if (threadIdx.x == 0) sm.count = 0;
    __syncthreads();
    const float low = bin < BINS - 1 ? sc.under(bin) : -INFINITY;  // (the last holds all further ones)
    items([&](float z, int i) {
        if (z >= low && sc.bin(z) == bin) {
            const uint32_t at = atomicAdd(&sm.count, 1u);
            if (int(at) < most) room[at] = item_of(z, i);
        }
    });
    __syncthreads();
    const int n = int(sm.count);
    if (n > most) return Cut::at(find_cut(items, sm, target, masses, w));
    return cut_in_bin(room, n, sm, left, masses, w);
}

// The cuts of top_k and top_p over items whose shares are summed by bins
// first; row_mass: the mass that top_p is a share of where it is known (0:
// it is summed here) and top_k is off; n: how many logits that mass is of,
// the items or a whole row that holds more.
template <typename S>
__device__ Cut cuts(S&& items, int n, const Settings& s, const Scale& sc, uint64_t row_mass, Shared& sm, uint64_t* room,
                    int most, const Weigh& w) {
    Cut cut;
#pragma unroll 1
    for (int step = s.k ? 0 : 1; step < (s.p < 1.0f ? 2 : 1); ++step) {
        const bool masses = step == 1;
        clear(sm.hist, BINS);
        uint64_t own = 0;
        // (atomics of many lanes on few bins cost more than exp: only what
        // the cut can reach is summed by bins)
        const int reach = masses && s.p > 0.0f ? sc.reach(s.p, 1.0f, n, s.t) : BINS - 1;
        items([&](float z, int i) {
            if (!cut.keeps(z, i)) return;
            const uint64_t v = masses ? w.mass(z) : 1;
            own += v;
            const int b = sc.bin(z);
            if (v && b <= reach) add(&sm.hist[b], v);
        });
        uint64_t target = uint64_t(s.k);
        if (masses) {
            const uint64_t total = block_sum(own, sm);
            target = share_of(s.p, row_mass && !s.k ? row_mass : total);
        }
        const Cut c = cut_by_bins(items, sc, sm, room, most, target, masses, w);
        if (c.z > cut.z || (c.z == cut.z && c.i < cut.i)) cut = c;
    }
    return cut;
}

// The exact cuts and the draw over the list's n items (every item that can
// be kept is there); `row_mass`: the mass that top_p is a share of, unless
// top_k is on, that of the row's sm.row_n logits.
__device__ void finish_list(int n, const Settings& s, float u, uint64_t row_mass, const Scale& sc, Shared& sm,
                            const Result& out) {
    const Weigh& w = out.w;
    const int tid = int(threadIdx.x);
    if (n <= PAIRS) {
        // Four threads an item: its place, the mass before it; the mass of
        // what stays; the running mass in index order.
        const int e = tid / 4, part = tid % 4;
        const uint64_t mine = e < n ? sm.item[e] : 0;
        const double x = e < n ? w(item_value(mine)) : 0.0;
        const uint64_t mass = Weigh::fixed(x);
        if (part == 0 && e < n) sm.mass[e] = mass;
        __syncthreads();
        uint64_t place = 0, before = 0;
        for (int j = part; j < n; j += 4) {
            if (sm.item[j] > mine) before += sm.mass[j], ++place;
        }
        place = quad_sum_u64(place), before = quad_sum_u64(before);
        bool keep = e < n && (s.k == 0 || place < uint64_t(s.k));
        if (s.p < 1.0f) {
            const uint64_t all = s.k ? block_sum(part == 0 && keep ? mass : 0, sm) : row_mass;
            keep = keep && before < share_of(s.p, all);
        }
        keep = keep && x >= s.least;
        if (part == 0 && e < n) sm.hist[e] = keep ? mass : 0;
        __syncthreads();
        uint64_t run = 0, total = 0;
        const int at = item_index(mine);
        for (int j = part; j < n; j += 4) {
            const uint64_t m = sm.hist[j];
            total += m;
            if (item_index(sm.item[j]) <= at) run += m;
        }
        run = quad_sum_u64(run), total = quad_sum_u64(total);
        const uint64_t target = goal(u, total);
        if (part == 0 && keep && mass > 0 && run >= target && run - mass < target)
            out.write(item_value(mine), at, total);
        return;
    }
    auto items = [&](auto&& f) {
#pragma unroll 1
        for (int i = tid; i < n; i += NT) f(item_value(sm.item[i]), item_index(sm.item[i]));
    };
    const Cut cut = cuts(items, s.k ? n : sm.row_n, s, sc, row_mass, sm, sm.edge, PAIRS, w);
    // the kept masses, then the draw: the digits of the index, 10 and 10 bits
    uint64_t own = 0;
#pragma unroll 1
    for (int i = tid; i < n; i += NT) {
        const float z = item_value(sm.item[i]);
        const double x = w(z);
        const uint64_t m = cut.keeps(z, item_index(sm.item[i])) && x >= s.least ? Weigh::fixed(x) : 0;
        sm.mass[i] = m;
        own += m;
    }
    const uint64_t total = block_sum(own, sm);
    uint64_t target = goal(u, total);
    int high = 0;
#pragma unroll 1
    for (int level = 0; level < 2; ++level) {
        clear(sm.hist, 1024);
#pragma unroll 1
        for (int i = tid; i < n; i += NT) {
            const int at = item_index(sm.item[i]);
            if (sm.mass[i] && (level == 0 || at >> 10 == high)) add(&sm.hist[level == 0 ? at >> 10 : at & 1023], sm.mass[i]);
        }
        pick<false>(sm.hist, 1024, target, sm);
        target -= sm.before;
        if (level == 0) high = int(sm.bin);
    }
    const int at = high << 10 | int(sm.bin);
    for (int i = tid; i < n; i += NT)
        if (item_index(sm.item[i]) == at) out.write(item_value(sm.item[i]), at, total);
}

// Gathers into the list the row's logits from `low` up, by the groups whose
// maxima reach it: the groups' numbers are collected first, so that four
// threads a group read them, two groups at a time in flight.  The count may
// pass CAP: then the list does not hold them all.
template <typename T>
__device__ int gather(const Row<T>& row, const float* groups, float low, Shared& sm) {
    uint32_t* ids = reinterpret_cast<uint32_t*>(sm.mass);
    constexpr int MOST = int(sizeof(sm.mass) / 4);  // (a row has up to 2^16 groups)
    static_assert(MOST == 16 * NT, "a turn over the groups' maxima fills the room for their numbers");
    const int ngroup = (row.n + GROUP - 1) / GROUP, tid = int(threadIdx.x);
    __syncthreads();
    if (tid == 0) sm.count = 0;
#pragma unroll 1
    for (int g0 = 0; g0 < ngroup; g0 += MOST) {
        __syncthreads();
        if (tid == 0) sm.bin = 0;
        // (four maxima a load, four loads under way)
        float4 m[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int g = g0 + (j * NT + tid) * 4;
            m[j] = *reinterpret_cast<const float4*>(groups + (g < ngroup ? g : 0));
        }
        __syncthreads();
        uint32_t in = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int g = g0 + (j * NT + tid) * 4;
            const uint32_t b = uint32_t(m[j].x >= low) | uint32_t(m[j].y >= low) << 1 | uint32_t(m[j].z >= low) << 2 |
                               uint32_t(m[j].w >= low) << 3;
            const int live = ngroup - g;  // (the room behind the last group's maximum)
            in |= (live >= 4 ? b : live > 0 ? b & ((1u << live) - 1) : 0u) << (4 * j);
        }
        int at = places(&sm.bin, __popc(in));
        for (uint32_t left = in; left; left &= left - 1) {
            const int b = __builtin_ctz(left);
            ids[at++] = uint32_t(g0 + (b / 4 * NT + tid) * 4 + b % 4);
        }
        __syncthreads();
        const int count = int(sm.bin), turns = (count + NT / 2 - 1) / (NT / 2);
#pragma unroll 1
        for (int t = 0; t < turns; ++t) {
            const int k = t * (NT / 2) + tid / 4, k2 = k + NT / 4;
            const int i0 = k < count ? int(ids[k]) * GROUP + tid % 4 * 4 : row.n;
            const int i1 = k2 < count ? int(ids[k2]) * GROUP + tid % 4 * 4 : row.n;
            const auto v0 = row.load(i0), v1 = row.load(i1);
            float z[8];
            row.four(v0, i0, z);
            row.four(v1, i1, z + 4);
            uint32_t pass = 0;
#pragma unroll
            for (int c = 0; c < 8; ++c) pass |= uint32_t(z[c] >= low) << c;
            int to = places(&sm.count, __popc(pass));
#pragma unroll
            for (int c = 0; c < 8; ++c)
                if (pass >> c & 1) {
                    if (to < CAP) sm.item[to] = item_of(z[c], (c < 4 ? i0 : i1) + c % 4);
                    ++to;
                }
        }
    }
    __syncthreads();
    return int(sm.count);
}

// From the counts of `units` maxima by bins, each of as many logits: the bin
// down to which the logits' mass is estimated to reach `target`, and their
// number (sm.found).  With c of the maxima at or above a threshold there are
// about -units log(1 - c / units) logits there.
__device__ inline int guess_bin(int units, uint64_t target, const Scale& sc, Shared& sm, const Weigh& w) {
    static_assert(BINS == 2 * NT, "two bins a thread");
    const int tid = int(threadIdx.x);
    __syncthreads();
    const uint64_t x0 = sm.hist[2 * tid], x1 = sm.hist[2 * tid + 1];
    const uint64_t scan = wave_scan_u64(x0 + x1);
    if (tid % WAVE == WAVE - 1) sm.part[wave_id()] = scan;
    __syncthreads();
    const uint64_t waves = row_scan_u64(sm.part[tid % NWAVE]);
    const uint64_t c2 = (wave_id() ? lane_u64(waves, wave_id() - 1) : 0) + scan, c1 = c2 - x1, c0 = c1 - x0;
    auto logits = [&](uint64_t c) {  // (saturated: more than any list holds)
        const float rest = 1.0f - float(c) / float(units);
        return rest > 0.0f ? -float(units) * __logf(rest) : 1e7f;
    };
    const float n0 = logits(c0), n1 = logits(c1), n2 = logits(c2);
    auto share = [&](float n, int bin) {
        return uint64_t(n > 0.0f ? double(n) * double(w.mass(sc.max - float(bin + 1) / sc.per)) : 0.0);
    };
    sm.hist[2 * tid] = share(n1 - n0, 2 * tid);
    sm.hist[2 * tid + 1] = share(n2 - n1, 2 * tid + 1);
    pick<false>(sm.hist, BINS, target, sm);
    const int bin = int(sm.bin);
    if (tid == bin / 2) sm.found = sm.total < target ? ~uint64_t(0) : uint64_t(bin % 2 ? n2 : n1);
    __syncthreads();
    return bin;
}

// The list that holds every token that the filters can keep, if one can be
// had: its length, or -1.  groups: the maxima of the row's groups; chunk: the
// thread's of its nchunk chunks (0: none are kept).
template <typename T>
__device__ int make_list(const Settings& s, const Scale& sc, Shared& sm, uint64_t row_mass, const Row<T>& row,
                         const float* groups, float chunk, int nchunk, const Weigh& w) {
    const bool by_p = s.k == 0 && s.least == 0.0;
    const int ngroup = (row.n + GROUP - 1) / GROUP;
    // top_p alone: a threshold with a little more mass above it by estimate,
    // then with more.
    const uint64_t want = by_p ? share_of(s.p, row_mass) : 0;
#pragma unroll 1
    for (int guess = w.infinite ? 2 : 0;; ++guess) {
        int last = -1;
        if (guess == 2) {
            // (everything)
        } else if (s.k || by_p) {
            // The coarsest maxima of which k are fewer than half: fewer
            // maxima to count, and hardly more logits above the k-th.
            const int k = s.k ? int(s.k) : ngroup >= 8192 ? ngroup / 8 : ngroup;
            clear(sm.hist, BINS);
            if (2 * k <= nchunk && s.k) {
                if (chunk > -INFINITY) add(&sm.hist[sc.bin(chunk)], 1);
            } else if (s.k && 2 * k > ngroup && row.n <= SHORT) {
                row.turns([&](const float* z, int) {
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        if (z[c] > -INFINITY) add(&sm.hist[sc.bin(z[c])], 1);
                });
            } else {
                const bool fours = 2 * k <= ngroup / 4;
#pragma unroll 2
                for (int g = int(threadIdx.x) * 4; g < ngroup; g += NT * 4) {
                    const float4 m = *reinterpret_cast<const float4*>(groups + g);
                    float x[4] = {m.x, g + 1 < ngroup ? m.y : -INFINITY, g + 2 < ngroup ? m.z : -INFINITY,
                                  g + 3 < ngroup ? m.w : -INFINITY};
                    if (fours) {
                        x[0] = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
                        if (x[0] > -INFINITY) add(&sm.hist[sc.bin(x[0])], 1);
                    } else {
#pragma unroll
                        for (int c = 0; c < 4; ++c)
                            if (x[c] > -INFINITY) add(&sm.hist[sc.bin(x[c])], 1);
                    }
                }
            }
            if (s.k) {
                pick<false>(sm.hist, BINS, uint64_t(k), sm);
                last = int(sm.bin);
            } else {
                const uint64_t rest = row_mass > want ? row_mass - want : 0;
                last = guess_bin(k < ngroup ? ngroup / 4 : ngroup, want + (guess == 0 ? rest / 4 : rest / 4 * 3), sc,
                                 sm, w);
                if (sm.found > PAIRS) return -1;  // (the wide kernels are no slower)
            }
        } else {
            last = sc.reach_min(s.least, s.t);
        }
        if (last == BINS - 1) last = sc.whole ? BINS - 2 : -1;  // (all that have a mass)
        const bool all = last < 0;
        if (all && row.n > CAP) return -1;
        const int n = gather(row, groups, all ? LOWEST : sc.under(last), sm);
        if (n <= CAP && (all || !by_p)) return n;
        if (n > CAP) return -1;
        uint64_t own = 0;
#pragma unroll 1
        for (int i = threadIdx.x; i < n; i += NT) own += w.mass(item_value(sm.item[i]));
        if (block_sum(own, sm) >= want) return n;
    }
}

// f(z, i, on) for a row's logits from `low` up (finite), 64 a wave at a time
// (on: the lane has one).  Few of a row's logits reach a cut, and some lane of
// a wave has one nearly always: without the lists each took the time of all,
// 8.5 us of exp for 16 a thread.
template <typename T, typename F>
__device__ inline void passing(const Row<T>& row, float low, Passed& list, F&& f) {
    float* lz = list.z[wave_id()];
    int* at = list.at[wave_id()];
    const int lane = int(threadIdx.x) % WAVE;
    int have = 0;
    const auto batch = [&](int from, bool on) {
        asm volatile("" ::: "memory");  // (a wave's LDS accesses are in order)
        f(on ? lz[from + lane] : -INFINITY, on ? at[from + lane] : 0, on);
        asm volatile("" ::: "memory");
    };
    row.turns([&](const float* z, int i) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const bool pass = z[c] >= low;
            const uint64_t all = __ballot(pass);
            if (!all) continue;
            if (pass) {
                const int to = have + int(__builtin_amdgcn_mbcnt_hi(uint32_t(all >> 32),
                                                                   __builtin_amdgcn_mbcnt_lo(uint32_t(all), 0)));
                lz[to] = z[c], at[to] = i + c;
            }
            have += __popcll(all);
        }
        for (; have >= WAVE; have -= WAVE) batch(have - WAVE, true);
    });
    if (have) batch(0, lane < have);
}

// A wave's masses m of logits i into the sums of their segments.
__device__ inline void add_segment(uint64_t* sums, int i, uint64_t m) {
    const int seg = i / SEG, one = __builtin_amdgcn_readfirstlane(seg);
    if (__all(seg == one)) {
        m = wave_scan_u64(m);
        if (threadIdx.x % WAVE == WAVE - 1 && m) add(&sums[one], m);
    } else if (m) {
        add(&sums[seg], m);
    }
}

// The exact cuts and the draw over a whole row whose kept tokens do not fit a
// list.
template <typename T>
__device__ void finish_row(const Row<T>& row, const Settings& s, float u, const Scale& sc, Shared& sm,
                           const Result& out) {
    auto items = [&](auto&& f) {
        row.turns([&](const float* z, int i) {
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (z[c] > -INFINITY) f(z[c], i + c);
        });
    };
    const Cut cut = cuts(items, row.n, s, sc, 0, sm, sm.item, CAP, out.w);
    auto kept = [&](float z, int i) -> uint64_t {
        if (!cut.keeps(z, i)) return 0;
        const double x = out.w(z);
        return x >= s.least ? Weigh::fixed(x) : 0;
    };
    const int ns = row.segments();
    __syncthreads();
    clear(sm.item, ns);
    passing(row, fmaxf(cut.z, LOWEST), sm.list, [&](float z, int i, bool on) { add_segment(sm.item, i, on ? kept(z, i) : 0); });
    __syncthreads();
    uint64_t own = 0;
    for (int i = threadIdx.x; i < ns; i += NT) own += sm.item[i];
    const uint64_t total = block_sum(own, sm), target = goal(u, total);
    pick<false>(sm.item, ns, target, sm);
    draw_in(row, int(sm.bin) * SEG, target - sm.before, total, out, kept);
}

// Long rows whose kept tokens do not fit a list, between the kernels.
enum Step : uint32_t { DONE = 0, TO_CUT, TO_DRAW, TO_FINISH };
struct Pending {
    uint64_t left;       // TO_CUT: the row's mass; TO_DRAW: what top_p takes from bin `bin`
    float max;
    uint32_t step;
    int bin;             // bins before it stay whole
    uint32_t arrived[2];
    uint32_t edges;      // logits of the bin
};
// What sample_stats leaves of CHUNK logits of a long row.
struct Chunk {
    float max;
    uint32_t first;  // index of the first maximum
    double sum;      // of exp((z - max) / T), where need_sum()
};
struct Workspace {
    Pending* pending;   // [rows]
    Chunk* chunks;      // [rows][nchunk] (this and what follows: long rows)
    float* groups;      // [rows][nchunk * CHUNK / GROUP]
    uint64_t* hist;     // [rows][nparts][BINS]
    uint64_t* segs;     // [rows][nchunk * CHUNK / SEG]
    uint64_t* edge;     // [rows][EDGE]
    int64_t nchunk, nparts;
    Workspace from(int64_t r) const {
        Workspace w = *this;
        w.pending += r, w.chunks += r * nchunk, w.groups += r * nchunk * (CHUNK / GROUP);
        w.hist += r * nparts * BINS, w.segs += r * nchunk * (CHUNK / SEG), w.edge += r * EDGE;
        return w;
    }
};

// Rows of at most SHORT logits: one workgroup a row.
template <typename T>
__global__ __launch_bounds__(NT) void sample_short(SampleArgs a) {
    __shared__ Shared sm;
    __shared__ __attribute__((aligned(16))) float groups[SHORT / GROUP];
    const int64_t r = blockIdx.x;
    const int tid = int(threadIdx.x);
    const Row<T> row(static_cast<const T*>(a.logits) + r * a.ld, a.vocab);
    const Settings s = settings_of(a, r);
    const float u = a.u[r];
    if (tid == 0) sm.kmax = 0, sm.kfirst = 0xffffffffu, sm.row_n = row.n;
    float zmax = -INFINITY;
    uint32_t first = 0xffffffffu;
    row.turns([&](const float* z, int i) {
        float m = fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3]));
        if (m > zmax) {
            zmax = m;
            first = uint32_t(i) + (z[0] == m ? 0 : z[1] == m ? 1 : z[2] == m ? 2 : 3);
        }
        m = fmaxf(m, dpp_f32<0xb1>(m));  // (four lanes of a quad: a group)
        m = fmaxf(m, dpp_f32<0x4e>(m));
        if (tid % 4 == 0 && i < SHORT) groups[i / GROUP] = m > -INFINITY ? m : -INFINITY;
    });
    const float wmax = wave_max(zmax);
    __syncthreads();
    if (tid % WAVE == 0 && wmax > -INFINITY) atomicMax(&sm.kmax, key_of(wmax));
    __syncthreads();
    const uint32_t kmax = __builtin_amdgcn_readfirstlane(sm.kmax);
    const float top = kmax ? value_of(kmax) : -INFINITY;
    const Result out(a, r, top, s);
    if (kmax == 0) {
        if (tid == 0) out.certain(-1);
        return;
    }
    if (s.greedy) {
        if (zmax == top) atomicMin(&sm.kfirst, first);
        __syncthreads();
        if (tid == 0) out.certain(int(sm.kfirst));
        return;
    }
    auto mass = [&](float z, int) { return out.w.mass(z); };
    const Scale sc(top, s.t);
    int n = -1;
    if (s.p >= 1.0f || s.k > 0 || s.least > 0.0) {  // (top_p alone: its masses by bins settle it in the fewest passes)
        uint64_t total = 0;
        if (s.need_sum()) {
            row.sums(sm.item, mass);
            __syncthreads();
            total = block_sum(tid < row.segments() ? sm.item[tid] : 0, sm);
            if (s.p >= 1.0f) {  // no filter
                const uint64_t target = goal(u, total);
                pick<false>(sm.item, row.segments(), target, sm);
                draw_in(row, int(sm.bin) * SEG, target - sm.before, total, out, mass);
                return;
            }
        }
        n = make_list(s, sc, sm, total, row, groups, -INFINITY, 0, out.w);
        if (n >= 0) finish_list(n, s, u, total, sc, sm, out);
    }
    if (n < 0) finish_row(row, s, u, sc, sm, out);
}

template <typename T, int VEC>
__global__ __launch_bounds__(256) void sample_stats(SampleArgs a, Workspace ws) {
    constexpr int L = CHUNK / WAVE / VEC, G = GROUP / VEC;  // loads of a lane; lanes of a group
    const int lane = int(threadIdx.x) % WAVE;
    const int64_t nchunk = ws.nchunk, id = int64_t(blockIdx.x) * 4 + wave_id();
    if (id >= a.rows * nchunk) return;
    const int64_t r = id / nchunk, c = id - r * nchunk;
    const T* p = static_cast<const T*>(a.logits) + r * a.ld + c * CHUNK;
    const int n = int(a.vocab - c * CHUNK < CHUNK ? a.vocab - c * CHUNK : CHUNK);
    float z[L][VEC];
    if (n == CHUNK) {
        typedef T vec __attribute__((ext_vector_type(VEC)));
        vec v[L];
#pragma unroll
        for (int j = 0; j < L; ++j) v[j] = *reinterpret_cast<const vec*>(p + (j * WAVE + lane) * VEC);
#pragma unroll
        for (int j = 0; j < L; ++j)
#pragma unroll
            for (int e = 0; e < VEC; ++e) z[j][e] = float(v[j][e]);
    } else {
#pragma unroll
        for (int j = 0; j < L; ++j)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const int i = (j * WAVE + lane) * VEC + e;
                z[j][e] = float(p[i < n ? i : n - 1]);
                if (i >= n) z[j][e] = -INFINITY;
            }
    }
    const Settings s = settings_of(a, r);
    float top = -INFINITY;
    float* gr = ws.groups + id * (CHUNK / GROUP);
#pragma unroll
    for (int j = 0; j < L; ++j) {
        float m = z[j][0];
#pragma unroll
        for (int e = 1; e < VEC; ++e) m = fmaxf(m, z[j][e]);
        top = fmaxf(top, m);
#pragma unroll
        for (int o = 1; o < G; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, WAVE));
        if (lane % G == 0) gr[(j * WAVE + lane) / G] = m > -INFINITY ? m : -INFINITY;
    }
    top = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, wave_max(top))));
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
        const Weigh w(top, s.inv_t);
#pragma unroll
        for (int j = 0; j < L; ++j)
#pragma unroll
            for (int e = 0; e < VEC; ++e) sum += w(z[j][e]);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, WAVE);
    }
    if (lane == 0) ws.chunks[id] = Chunk{top, first, sum};
}

template <typename T>
__global__ __launch_bounds__(NT) void sample_long(SampleArgs a, Workspace ws) {
    __shared__ Shared sm;
    const int64_t r = blockIdx.x;
    const int tid = int(threadIdx.x), nchunk = int(ws.nchunk);  // (nchunk <= NT)
    const Chunk mine = tid < nchunk ? ws.chunks[r * nchunk + tid] : Chunk{-INFINITY, 0xffffffffu, 0.0};
    const Settings s = settings_of(a, r);
    const float u = a.u[r];
    const float* groups = ws.groups + r * nchunk * (CHUNK / GROUP);
    const Row<T> row(static_cast<const T*>(a.logits) + r * a.ld, a.vocab);
    if (tid == 0) sm.kmax = 0, sm.kfirst = 0xffffffffu, sm.row_n = row.n, ws.pending[r].step = DONE;
    const float wmax = wave_max(mine.max);
    __syncthreads();
    if (tid % WAVE == 0 && wmax > -INFINITY) atomicMax(&sm.kmax, key_of(wmax));
    __syncthreads();
    const uint32_t kmax = __builtin_amdgcn_readfirstlane(sm.kmax);
    const float top = kmax ? value_of(kmax) : -INFINITY;
    const Result out(a, r, top, s);
    if (kmax == 0) {
        if (tid == 0) out.certain(-1);
        return;
    }
    if (s.greedy) {
        if (mine.max == top) atomicMin(&sm.kfirst, mine.first);
        __syncthreads();
        if (tid == 0) out.certain(int(sm.kfirst));
        return;
    }
    uint64_t total = 0;
    if (s.need_sum()) {
        // (a chunk has a mass where one of its logits has)
        const double x = out.w(mine.max);
        const uint64_t own = Weigh::fixed(x) ? uint64_t(rint(mine.sum * x * ONE)) : 0;
        total = block_sum(own, sm);
        if (s.p >= 1.0f) {  // no filter: the chunk, its segment, the logit
            sm.hist[tid] = own;
            const uint64_t target = goal(u, total);
            pick<false>(sm.hist, NT, target, sm);
            const int c = int(sm.bin);
            const uint64_t left = target - sm.before;
            const Row<T> part(row.p + c * CHUNK, row.n - c * CHUNK < CHUNK ? row.n - c * CHUNK : CHUNK);
            auto mass = [&](float z, int) { return out.w.mass(z); };
            __syncthreads();
            part.sums(sm.item, mass);
            pick<false>(sm.item, part.segments(), left, sm);
            // (the chunk's sum and its logits' masses differ by their
            // rounding: past the end is the last logit with a mass)
            int seg = int(sm.bin);
            uint64_t rest = left > sm.before ? left - sm.before : 1;
            if (sm.total < left) {
                while (seg > 0 && sm.item[seg] == 0) --seg;
                rest = sm.item[seg];
            }
            draw_in(row, c * CHUNK + seg * SEG, rest, total, out, mass);
            return;
        }
    }
    const Scale sc(top, s.t);
    const int n = make_list(s, sc, sm, total, row, groups, mine.max, nchunk, out.w);
    if (n >= 0) {
        finish_list(n, s, u, total, sc, sm, out);
        return;
    }
    if (tid == 0)
        ws.pending[r] = Pending{total, top, s.k ? TO_FINISH : s.p < 1.0f ? TO_CUT : TO_DRAW, BINS, {0, 0}, 0};
}

// Long rows TO_FINISH (in sample_long their pass's registers slowed the lists
// of the others: 256 rows of 128,257 132 -> 135 us).
template <typename T>
__global__ __launch_bounds__(NT) void sample_row(SampleArgs a, Workspace ws) {
    const int64_t r = blockIdx.x;
    const Pending& pd = ws.pending[r];
    if (pd.step != TO_FINISH) return;
    __shared__ Shared sm;
    const Settings s = settings_of(a, r);
    const Row<T> row(static_cast<const T*>(a.logits) + r * a.ld, a.vocab);
    finish_row(row, s, a.u[r], Scale(pd.max, s.t), sm, Result(a, r, pd.max, s));
}

// Whether this workgroup is the last of its row's to arrive; what the others
// left for it, by store_shared, is then there for load_shared.  These go past
// the L2s, which are one an XCD: the stores are done when they are waited
// for, and no fence, which would write back and invalidate an L2, is needed
// (one a workgroup took 50 us of a pass over 16.8 million logits, one a wave
// 300).  This relies on the hardware and not on the language's memory model,
// which orders relaxed accesses to different places by fences alone: on gfx950
// stores and loads of agent scope carry sc1, and a store has left vmcnt when
// other XCDs can read it.  The barrier has every wave's wait before the one
// add; the loads follow the add's return, which the second barrier waits for.
__device__ inline bool last_of(uint32_t* arrived, Common& sm) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0)
        sm.count = __hip_atomic_fetch_add(arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    const bool last = sm.count == gridDim.x - 1;
    __syncthreads();
    return last;
}
__device__ inline void store_shared(uint64_t* p, uint64_t v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ inline uint64_t load_shared(const uint64_t* p) {  // written by other workgroups of this launch
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The logits of this workgroup's part of a row.
template <typename T>
__device__ inline Row<T> part_of(const Row<T>& row) {
    const int first = int(blockIdx.x) * PART;
    return Row<T>(row.p + first, row.n - first < PART ? row.n - first : PART);
}

// The masses of rows TO_CUT by bins; the last workgroup of a row finds
// top_p's cut.
template <typename T>
__global__ __launch_bounds__(NT, 8) void sample_bins(SampleArgs a, Workspace ws) {
    const int64_t r = blockIdx.y;
    Pending& pd = ws.pending[r];
    if (pd.step != TO_CUT) return;
    __shared__ BinsShared sm;
    const int tid = int(threadIdx.x);
    const Settings s = settings_of(a, r);
    const Row<T> row(static_cast<const T*>(a.logits) + r * a.ld, a.vocab);
    const Weigh w(pd.max, s.inv_t);
    const Scale sc(pd.max, s.t);
    const uint64_t total = pd.left;
    const int reach = s.p > 0.0f ? sc.reach(s.p, float(double(total) / ONE), row.n, s.t) : BINS - 1;
    clear(sm.hist, BINS);
    passing(part_of(row), sc.low(reach), sm.list, [&](float z, int, bool on) {
        const int b = sc.bin(z);
        const uint64_t m = on && b <= reach ? w.mass(z) : 0;
        if (m) add(&sm.hist[b], m);
    });
    __syncthreads();
    uint64_t* hist = ws.hist + r * ws.nparts * BINS;
    for (int i = tid; i <= reach; i += NT) store_shared(hist + blockIdx.x * BINS + i, sm.hist[i]);
    if (!last_of(&pd.arrived[0], sm)) return;
#pragma unroll
    for (int i = tid; i < BINS; i += NT) {
        uint64_t v = 0;
        if (i <= reach) {
#pragma unroll 8
            for (int k = 0; k < int(ws.nparts); ++k) v += load_shared(hist + k * BINS + i);
        }
        sm.hist[i] = v;
    }
    const uint64_t target = share_of(s.p, total);
    pick<false>(sm.hist, BINS, target, sm);
    if (tid == 0) pd.bin = int(sm.bin), pd.left = target - sm.before, pd.step = TO_DRAW;
}

// The kept masses of rows TO_DRAW by segments, the logits of the bin that
// top_p cuts set apart; the last workgroup of a row cuts and draws.
template <typename T>
__global__ __launch_bounds__(NT, 8) void sample_draw(SampleArgs a, Workspace ws) {
    const int64_t r = blockIdx.y;
    Pending& pd = ws.pending[r];
    if (pd.step != TO_DRAW) return;
    __shared__ DrawShared sm;
    const int tid = int(threadIdx.x), bin = pd.bin;
    const Settings s = settings_of(a, r);
    const Row<T> row(static_cast<const T*>(a.logits) + r * a.ld, a.vocab);
    const Result out(a, r, pd.max, s);
    const Scale sc(pd.max, s.t);
    const int first = int(blockIdx.x) * PART, ns = row.segments();
    uint64_t* segs = ws.segs + r * ws.nchunk * (CHUNK / SEG);
    uint64_t* edge = ws.edge + r * EDGE;
    const Row<T> part = part_of(row);
    if (tid == 0) sm.count = 0;
    if (tid < PART / SEG) sm.seg[tid] = 0;
    __syncthreads();
    // (a logit in a bin before stays, if min_p lets it)
    const int last = s.least > 0.0 ? sc.reach_min(s.least, s.t) : BINS;
    passing(part, sc.low(bin < last ? bin : last), sm.list, [&](float z, int i, bool on) {
        const int b = on ? sc.bin(z) : BINS;
        if (b == bin && on) {
            const uint32_t at = atomicAdd(&sm.count, 1u);
            if (at < EDGE) sm.edge[at] = item_of(z, first + i);
        }
        uint64_t m = 0;
        if (b < bin) {
            const double x = out.w(z);
            m = x >= s.least ? Weigh::fixed(x) : 0;
        }
        add_segment(sm.seg, i, m);
    });
    __syncthreads();
    const uint32_t here = sm.count;
    if (tid == 0 && here) sm.bin = atomicAdd(&pd.edges, here);
    __syncthreads();
    for (uint32_t i = tid; i < here && sm.bin + i < EDGE; i += NT)
        store_shared(edge + sm.bin + i, sm.edge[i]);
    if (tid < part.segments())
        store_shared(segs + first / SEG + tid, sm.seg[tid]);
    if (!last_of(&pd.arrived[1], sm)) return;
    if (tid == 0) sm.kfirst = __hip_atomic_load(&pd.edges, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    for (int i = tid; i < ns; i += NT) sm.item[i] = load_shared(segs + i);
    __syncthreads();
    const int n = int(sm.kfirst);
    Cut cut;
    if (n > 0 && n <= EDGE) {
        for (int i = tid; i < n; i += NT) sm.edge[i] = load_shared(edge + i);
        cut = cut_in_bin(sm.edge, n, sm, pd.left, true, out.w);
    } else if (n > EDGE) {
        auto items = [&](auto&& f) {
            row.turns([&](const float* z, int i) {
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (z[c] > -INFINITY && sc.bin(z[c]) == bin) f(z[c], i + c);
            });
        };
        cut = Cut::at(find_cut(items, sm, pd.left, true, out.w));
    }
    // (an edge that is no item may lie below the bin: both conditions hold)
    auto kept = [&](float z, int i) -> uint64_t {
        if (sc.bin(z) > bin || !cut.keeps(z, i)) return 0;
        const double x = out.w(z);
        return x >= s.least ? Weigh::fixed(x) : 0;
    };
    if (n <= EDGE) {
        for (int i = tid; i < n; i += NT) {
            const uint64_t m = kept(item_value(sm.edge[i]), item_index(sm.edge[i]));
            if (m) add(&sm.item[item_index(sm.edge[i]) / SEG], m);
        }
    } else {
        __syncthreads();
        row.sums(sm.item, kept);
    }
    __syncthreads();
    uint64_t own = 0;
    for (int i = tid; i < ns; i += NT) own += sm.item[i];
    const uint64_t total = block_sum(own, sm), target = goal(a.u[r], total);
    pick<false>(sm.item, ns, target, sm);
    draw_in(row, int(sm.bin) * SEG, target - sm.before, total, out, kept);
}

void check(const SampleArgs& a) {
    if (a.dtype != ELEM_F32 && a.dtype != ELEM_F16 && a.dtype != ELEM_BF16)
        fail(E_INVALID, "sample: logits must be f32, f16 or bf16");
    if (a.rows <= 0 || a.rows > (1 << 21)) fail(E_INVALID, "sample: rows must be 1 to 2^21");
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

int64_t chunks_of(int64_t vocab) { return vocab <= SHORT ? 0 : (vocab + CHUNK - 1) / CHUNK; }

int64_t parts_of(int64_t vocab) { return (vocab + PART - 1) / PART; }

template <typename T>
void launch(hipStream_t s, const SampleArgs& a, void* workspace) {
    const dim3 grid{unsigned(a.rows)}, block{NT};
    if (a.vocab <= SHORT) {
        sample_short<T><<<grid, block, 0, s>>>(a);
        OMG_HIP(hipGetLastError());
        return;
    }
    Workspace ws{};
    ws.nchunk = chunks_of(a.vocab);
    ws.nparts = parts_of(a.vocab);
    const int64_t n = a.rows * ws.nchunk;
    ws.pending = static_cast<Pending*>(workspace);
    ws.chunks = reinterpret_cast<Chunk*>(ws.pending + a.rows);
    ws.groups = reinterpret_cast<float*>(ws.chunks + n);
    ws.hist = reinterpret_cast<uint64_t*>(ws.groups + n * (CHUNK / GROUP));
    ws.segs = ws.hist + a.rows * ws.nparts * BINS;
    ws.edge = ws.segs + n * (CHUNK / SEG);
    if ((n + 3) / 4 >= MAX_BLOCKS) fail(E_CAPACITY, "sample: too many logits for one call");
    const dim3 wide{unsigned((n + 3) / 4)};
    constexpr int VEC = 16 / int(sizeof(T));
    if (reinterpret_cast<uintptr_t>(a.logits) % 16 == 0 && a.ld % VEC == 0)
        sample_stats<T, VEC><<<wide, dim3(256), 0, s>>>(a, ws);
    else
        sample_stats<T, 1><<<wide, dim3(256), 0, s>>>(a, ws);
    OMG_HIP(hipGetLastError());
    sample_long<T><<<grid, block, 0, s>>>(a, ws);
    OMG_HIP(hipGetLastError());
    if (a.top_k) {
        sample_row<T><<<grid, block, 0, s>>>(a, ws);
        OMG_HIP(hipGetLastError());
    }
    if (!a.top_p && !a.min_p) return;
    for (int64_t r = 0; r < a.rows; r += 65535) {  // (a grid's second size)
        const dim3 parts{unsigned(ws.nparts), unsigned(std::min<int64_t>(65535, a.rows - r))};
        if (a.top_p) sample_bins<T><<<parts, block, 0, s>>>(rows_from<T>(a, r), ws.from(r));
        OMG_HIP(hipGetLastError());
        sample_draw<T><<<parts, block, 0, s>>>(rows_from<T>(a, r), ws.from(r));
        OMG_HIP(hipGetLastError());
    }
}

}  // namespace

int64_t sample_workspace(int64_t rows, int64_t vocab) {
    SampleArgs a{};
    a.rows = rows, a.vocab = vocab;
    check(a);
    static_assert(sizeof(Pending) % 16 == 0 && sizeof(Chunk) % 16 == 0, "the workspace's arrays are aligned");
    const int64_t n = chunks_of(vocab);
    if (n == 0) return 0;
    return rows * (int64_t(sizeof(Pending)) + n * int64_t(sizeof(Chunk) + CHUNK / SEG * 8 + CHUNK / GROUP * 4) +
                   parts_of(vocab) * BINS * 8 + EDGE * 8);
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
