// Device helpers of the paged-cache and sampling kernels: element types,
// 8-wide loads and stores, and the sequence a token row belongs to.
#pragma once

#include "kern_common.h"

namespace omg {

constexpr int64_t MAX_BLOCKS = 1 << 24;  // of 256 threads: a launch holds less than 2^32 threads

// Host checks of the descriptions, shared by the calls that take them (paged.hip).
bool aligned16(const void* p);
int log2_of(int64_t n);  // the least s with 2^s >= n
void check_kv(const PagedKv& kv, const char* who);
void check_batch(const PagedBatch& b, const PagedKv& kv, const char* who);

typedef __bf16 bf16_t;
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));

template <typename T>
struct Vec8;
template <>
struct Vec8<half_t> {
    typedef half8 type;
};
template <>
struct Vec8<bf16_t> {
    typedef bf16x8 type;
};

// Eight consecutive elements as f32 (16-byte aligned).
template <typename T>
__device__ inline void load8(const T* p, float* x) {
    if constexpr (sizeof(T) == 4) {
        const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
        x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
        const typename Vec8<T>::type v = *reinterpret_cast<const typename Vec8<T>::type*>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = float(v[i]);
    }
}

// Eight values rounded to nearest even (16-byte aligned).
template <typename T>
__device__ inline void store8(T* p, const float* x) {
    typename Vec8<T>::type v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = T(x[i]);
    *reinterpret_cast<typename Vec8<T>::type*>(p) = v;
}

// How many of a[1..n] (not descending) are at most `x`; every lane of the
// wave calls it with the same arguments but its own lane: 64 probes a step.
__device__ inline int64_t count_le(const int32_t* a, int64_t n, int64_t x, int lane) {
    int64_t lo = 0;
    while (n > 0) {
        const int64_t step = (n + WAVE - 1) / WAVE, i = lo + (lane + 1) * step;
        const int c = __popcll(__ballot(i <= lo + n && a[i <= lo + n ? i : lo + n] <= x));
        const int64_t rest = n - c * step;
        lo += c * step;
        n = rest < step - 1 ? rest : step - 1;
    }
    return lo;
}

// The sequence of a token row (-1: none) and its row in the sequence's own
// cache rows (below 0 where lens[seq] leaves no room for it).
struct SeqRow {
    int64_t seq, row;
};
__device__ inline SeqRow token_row(const PagedBatch& b, int64_t tok, int lane) {
    if (!b.start) return {tok, int64_t(b.lens[tok]) - 1};
    const int64_t s = count_le(b.start, b.nseq, tok, lane);
    if (s >= b.nseq || tok < b.start[0]) return {-1, 0};
    return {s, int64_t(b.lens[s]) - (int64_t(b.start[s + 1]) - tok)};
}

}  // namespace omg
