// Sampling the next token from rows of logits (omg_dev_sample).
//
// A token is kept or not by its place in the order (z descending, index
// ascending), so what a filter keeps is a threshold: every z above it and
// the first `ties` tokens equal to it.  Masses are sums of
//   W(z) = round(2^42 exp((z - max) / T)),
// whole numbers that add up the same in any order (at most 2^20 of them, so
// 2^62): the histograms' atomics and the split of a row over threads leave
// no trace in the result.  exp is taken in 64 bits.
#include <string>

#include "common.h"
#include "kern_common.h"
#include "paged.h"

namespace omg {

namespace {

constexpr int NT = 1024;  // threads of a row's workgroup
constexpr int DIG = 2048; // histogram bins: the key's digits are 11, 11 and 10 bits

// Order-preserving bits of a logit; 0 for masked ones (-infinity, NaN).
// (z + 0 makes -0 the 0 it equals.)
__device__ inline uint32_t key_of(float z) {
    if (!(z > -INFINITY)) return 0;
    const uint32_t u = __builtin_bit_cast(uint32_t, z + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ inline float value_of(uint32_t k) {
    return __builtin_bit_cast(float, k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// What stays of a row: keys above `key`, and the first `ties` equal to it.
struct Cut {
    uint32_t key;
    uint64_t ties;
};

struct Shared {
    uint64_t hist[DIG];
    uint64_t part[NT / WAVE], part2[NT / WAVE];
    uint64_t found, before;
    uint32_t bin;
    uint32_t kmax, kfirst;
};

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

template <typename T>
struct RowOf {
    const T* z;
    int64_t n;
    double max, inv_t;  // (inv_t unused for an infinite maximum)
    __device__ uint32_t key(int64_t i) const { return key_of(float(z[i])); }
    // exp((z - max) / T): 1 at the maximum, whatever it is
    __device__ double weight(uint32_t k) const {
        if (k == 0) return 0.0;
        const double d = double(value_of(k)) - max;
        if (!(d < 0.0)) return 1.0;  // (infinity - infinity)
        const double x = d * inv_t;
        return x > -40.0 ? exp(x) : 0.0;
    }
    __device__ uint64_t mass(uint32_t k) const { return uint64_t(rint(weight(k) * 4398046511104.0)); }
};

// Sum of v over the workgroup, in every thread.
__device__ inline uint64_t block_sum(uint64_t v, uint64_t* part) {
    const int lane = int(threadIdx.x) % WAVE, wave = int(threadIdx.x) / WAVE;
    v = wave_sum_u64(v);
    __syncthreads();
    if (lane == 0) part[wave] = v;
    __syncthreads();
    uint64_t s = 0;
    for (int i = 0; i < NT / WAVE; ++i) s += part[i];
    return s;
}

// The element at which the running sum, over keys from the largest down,
// first reaches `target` (at least 1): `what` gives each key's share (a count
// of one, or its mass) and `limit` the keys that take part.  Returns its key
// and how many of the keys equal to it are needed.
template <typename T, typename F>
__device__ Cut find_cut(const RowOf<T>& row, Shared& sm, uint64_t target, const Cut& limit, F&& what) {
    uint32_t prefix = 0;
    uint64_t before = 0;
    for (int level = 0; level < 3; ++level) {
        const int shift = level == 0 ? 21 : level == 1 ? 10 : 0, bits = level == 2 ? 10 : 11;
        __syncthreads();
        for (int i = threadIdx.x; i < DIG; i += NT) sm.hist[i] = 0;
        __syncthreads();
        for (int64_t i = threadIdx.x; i < row.n; i += NT) {
            const uint32_t k = row.key(i);
            if (k <= limit.key || (level > 0 && (k >> (shift + bits)) != prefix)) continue;
            atomicAdd(reinterpret_cast<unsigned long long*>(&sm.hist[(k >> shift) & ((1u << bits) - 1)]),
                      static_cast<unsigned long long>(what(k)));
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            if (limit.key && limit.ties && (level == 0 || (limit.key >> (shift + bits)) == prefix))
                sm.hist[(limit.key >> shift) & ((1u << bits) - 1)] += limit.ties * what(limit.key);
            uint64_t run = before;
            uint32_t b = (1u << bits) - 1;
            for (;; --b) {
                if (run + sm.hist[b] >= target || b == 0) break;
                run += sm.hist[b];
            }
            sm.bin = b;
            sm.before = run;
        }
        __syncthreads();
        prefix = (prefix << bits) | sm.bin;
        before = sm.before;
    }
    const uint64_t one = what(prefix);
    return {prefix, one ? (target - before + one - 1) / one : 1};
}

template <typename T>
__global__ __launch_bounds__(NT) void sample_kernel(SampleArgs a) {
    __shared__ Shared sm;
    const int64_t r = blockIdx.x;
    const int tid = int(threadIdx.x), lane = tid % WAVE, wave = tid / WAVE;
    RowOf<T> row{static_cast<const T*>(a.logits) + r * a.ld, a.vocab, 0.0, 0.0};
    const float temp = a.temperature ? a.temperature[r] : 1.0f;

    // The maximum and its first index.
    if (tid == 0) sm.kmax = 0, sm.kfirst = 0xffffffffu;
    __syncthreads();
    uint32_t kmax = 0, at = 0xffffffffu;
    for (int64_t i = tid; i < row.n; i += NT) {
        const uint32_t k = row.key(i);
        if (k > kmax) kmax = k, at = uint32_t(i);
    }
    atomicMax(&sm.kmax, kmax);
    __syncthreads();
    if (kmax == sm.kmax) atomicMin(&sm.kfirst, at);
    __syncthreads();
    kmax = sm.kmax;
    if (kmax == 0 || !(temp > 0.0f)) {
        if (tid == 0) {
            a.tokens[r] = kmax == 0 ? -1 : int32_t(sm.kfirst);
            if (a.logprob) a.logprob[r] = kmax == 0 ? -INFINITY : 0.0f;
        }
        return;
    }
    row.max = double(value_of(kmax));
    row.inv_t = 1.0 / double(temp);

    Cut cut{0, 0};  // everything that is not masked
    const int64_t k = a.top_k ? int64_t(a.top_k[r]) : 0;
    if (k > 0 && k < row.n) cut = find_cut(row, sm, uint64_t(k), cut, [](uint32_t) { return uint64_t(1); });
    const float p = a.top_p ? a.top_p[r] : 1.0f;
    if (p < 1.0f) {
        uint64_t own = 0;
        for (int64_t i = tid; i < row.n; i += NT) {
            const uint32_t q = row.key(i);
            if (q > cut.key) own += row.mass(q);
        }
        const uint64_t total = block_sum(own, sm.part) + (cut.key ? cut.ties * row.mass(cut.key) : 0);
        const double want = ceil(double(p) * double(total));
        const uint64_t target = want < 1.0 ? 1 : uint64_t(want);
        cut = find_cut(row, sm, target < total ? target : total, cut,
                       [&](uint32_t q) { return row.mass(q); });
    }
    const float mp = a.min_p ? a.min_p[r] : 0.0f;
    const double least = mp > 0.0f ? (mp < 1.0f ? double(mp) : 1.0) : 0.0;

    // The kept masses in index order: ranges of the row, one per wave, then
    // the range that holds the drawn token in 16 again, down to one element
    // a lane.
    auto kept_mass = [&](uint32_t q) -> uint64_t {
        return least > 0.0 && row.weight(q) < least ? 0 : row.mass(q);
    };
    const uint64_t tie_mass = cut.key ? kept_mass(cut.key) : 0;
    int64_t lo = 0, n = row.n;
    uint64_t ties_before = 0, target = 0, total = 0;
    for (int level = 0;; ++level) {
        const int64_t span = (n + NT / WAVE - 1) / (NT / WAVE);
        const int64_t b = lo + wave * span, e = b + span < lo + n ? b + span : lo + n;
        uint64_t above = 0, ties = 0;
        for (int64_t i = b + lane; i < e; i += WAVE) {
            const uint32_t q = row.key(i);
            if (q > cut.key) above += kept_mass(q);
            if (q == cut.key && cut.key) ++ties;
        }
        above = wave_sum_u64(above);
        ties = wave_sum_u64(ties);
        __syncthreads();
        if (lane == 0) sm.part[wave] = above, sm.part2[wave] = ties;
        __syncthreads();
        // every thread runs over the 16 ranges
        auto range_mass = [&](int i, uint64_t& seen) {
            const uint64_t left = cut.ties > seen ? cut.ties - seen : 0;
            const uint64_t use = sm.part2[i] < left ? sm.part2[i] : left;
            seen += sm.part2[i];
            return sm.part[i] + use * tie_mass;
        };
        if (level == 0) {
            uint64_t seen = 0;
            for (int i = 0; i < NT / WAVE; ++i) total += range_mass(i, seen);
            const float u = a.u[r];
            const double t = (u > 0.0f ? (u < 1.0f ? double(u) : 1.0) : 0.0) * double(total);
            target = uint64_t(t) + 1;  // the first running mass > u total
            if (target > total) target = total;
        }
        uint64_t seen = ties_before, run = 0;
        int pick = 0;
        for (; pick < NT / WAVE; ++pick) {
            const uint64_t s0 = seen;
            const uint64_t m = range_mass(pick, seen);
            if (run + m >= target) {
                seen = s0;
                break;
            }
            run += m;
        }
        target -= run;
        ties_before = seen;
        lo += pick * span;
        n = n - pick * span < span ? n - pick * span : span;
        if (n <= WAVE) break;
    }
    if (wave == 0) {
        const uint32_t q = lane < n ? row.key(lo + lane) : 0;
        const uint64_t mine = q == cut.key && cut.key ? 1 : 0;
        const uint64_t rank = ties_before + wave_scan_u64(mine, lane);
        const uint64_t m = q > cut.key ? kept_mass(q) : mine && rank <= cut.ties ? tie_mass : 0;
        const uint64_t run = wave_scan_u64(m, lane);
        const uint64_t hit = __ballot(run >= target && m > 0);
        if (hit && lane == __builtin_ctzll(hit)) {
            a.tokens[r] = int32_t(lo + lane);
            const double d = double(value_of(q)) - row.max;
            if (a.logprob) a.logprob[r] = float((d < 0.0 ? d * row.inv_t : 0.0) - log(double(total) / 4398046511104.0));
        }
    }
}

void check(const SampleArgs& a) {
    if (a.dtype != ELEM_F32 && a.dtype != ELEM_F16 && a.dtype != ELEM_BF16)
        fail(E_INVALID, "sample: logits must be f32, f16 or bf16");
    if (a.rows <= 0 || a.rows > (1 << 24)) fail(E_INVALID, "sample: rows must be 1 to 2^24");
    if (a.vocab <= 0 || a.vocab > (1 << 20)) fail(E_INVALID, "sample: vocab must be 1 to 2^20");
}

}  // namespace

int64_t sample_workspace(int64_t rows, int64_t vocab) {
    SampleArgs a{};
    a.rows = rows, a.vocab = vocab;
    check(a);
    return 0;
}

void launch_sample(hipStream_t s, const SampleArgs& a, void* workspace, size_t bytes) {
    check(a);
    if (a.ld < a.vocab) fail(E_INVALID, "sample: ld must hold the vocabulary");
    if (!a.logits || !a.u || !a.tokens) fail(E_INVALID, "sample: null logits, u or tokens");
    if (reinterpret_cast<uintptr_t>(a.logits) % (a.dtype == ELEM_F32 ? 4 : 2))
        fail(E_INVALID, "sample: logits must be aligned to their type");
    const dim3 grid{unsigned(a.rows)}, block{NT};
    if (a.dtype == ELEM_F32)
        sample_kernel<float><<<grid, block, 0, s>>>(a);
    else if (a.dtype == ELEM_F16)
        sample_kernel<half_t><<<grid, block, 0, s>>>(a);
    else
        sample_kernel<bf16_t><<<grid, block, 0, s>>>(a);
    OMG_HIP(hipGetLastError());
}

}  // namespace omg
