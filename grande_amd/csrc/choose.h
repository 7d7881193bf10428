// The `left` largest of n values, in the order of their places: one workgroup
// of T threads a list.
//
// Values become 32-bit keys of the same order.  Passes over 8 bits each, from
// the top, narrow the key of the last one chosen down (a histogram of 256 bins,
// 8 copies by lane, so that equal bits seldom meet in one LDS word) until at
// most FEW values share the bits found: these are counted against each other.
// Then a pass counts per 64 values what lies over that key and at it, and a last
// one hands out the chosen, of the equal ones the first.  A chain of barriers:
// with HELD, up to R T values stay in registers; others are read again from L2
// in each pass.  (126 values by 256 threads 5 to 6 us, 1,050 9 us, 2,300 by 1,024
// threads 9.6 us, launch and all.)
#pragma once

#include "paged.h"

namespace omg {

constexpr int CHOOSE_R = 8;  // values of a thread in registers

// Ascending with the value; NaN lowest, the zeros alike.
__device__ inline uint32_t value_key(float w) {
    const uint32_t u = __builtin_bit_cast(uint32_t, w + 0.0f);
    return w != w ? 0u : u >> 31 ? ~u : u | 0x80000000u;
}

template <int T, bool HELD>
struct Choose {
    static constexpr int R = CHOOSE_R, WAVES = T / WAVE;
    static constexpr int CELLS = T;  // of 64 values: a part of the list
    static constexpr int COPIES = 8, FEW = 128;
    static_assert(T >= 256 && T % 256 == 0, "a thread a bin");
    struct Shared {
        alignas(16) uint32_t bins[COPIES * 256];
        uint32_t cells[2 * CELLS];
        uint32_t few[FEW], sums[2 * (WAVES < 4 ? 4 : WAVES)], found[3], nfew;
    };

    // The same for n <= T values, one a thread: how many lie over it, and of equal
    // ones before it, says whether it is chosen.
    template <typename F>
    static __device__ void run_few(Shared& sh, float value, int n, uint32_t left, F hand) {
        static_assert(T <= COPIES * 256);
        const int tid = int(threadIdx.x), lane = tid % WAVE, wave = __builtin_amdgcn_readfirstlane(tid / WAVE);
        const uint32_t key = tid < n ? value_key(value) : 0;
        const uint64_t before = (uint64_t(1) << lane) - 1;
        sh.bins[tid] = key;
        __syncthreads();
        uint32_t order = 0;
        for (int i = 0; i * WAVE < n; ++i) {  // (the keys behind the last one are over none and before none)
            const uint4* cell = reinterpret_cast<const uint4*>(sh.bins + i * WAVE);
            const uint32_t least = i < wave ? key : key + 1;  // (no key is 2^32 - 1)
#pragma unroll
            for (int j = 0; j < WAVE / 4; ++j) {
                const uint4 k = cell[j];
                order += (k.x >= least) + (k.y >= least) + (k.z >= least) + (k.w >= least);
            }
        }
        uint64_t like = 0;  // the wave's
#pragma unroll
        for (int j = 0; j < WAVE; ++j) like |= uint64_t(uint32_t(__builtin_amdgcn_readlane(int(key), j)) == key) << j;
        order += __popcll(like & before);
        const uint64_t chosen = __ballot(tid < n && order < left);
        if (lane == 0) sh.sums[wave] = __popcll(chosen);
        __syncthreads();
        int rank = __popcll(chosen & before);
        for (int i = 0; i < wave; ++i) rank += sh.sums[i];
        if (tid < n && order < left) hand(rank, tid, value);
        __syncthreads();
    }

    // hand(rank, place, value) for each chosen one of w[0 .. n), left <= n; the
    // list may be overwritten from its start on as they are handed out (a
    // chosen value's rank is at most its place, and all are read before).
    template <typename F>
    static __device__ void run(Shared& sh, const float* w, int n, uint32_t left, F hand) {
        const int tid = int(threadIdx.x), lane = tid % WAVE, wave = __builtin_amdgcn_readfirstlane(tid / WAVE);
        float held[R];
        if constexpr (HELD) {
#pragma unroll
            for (int u = 0; u < R; ++u) held[u] = tid + u * T < n ? w[tid + u * T] : 0.0f;
        }
        // f(key) for each of the thread's values.
        auto each = [&](auto f) {
            if constexpr (HELD) {
#pragma unroll
                for (int u = 0; u < R; ++u)  // (a branch of the wave, then one of its lanes)
                    if (wave * WAVE + u * T < n && tid + u * T < n) f(value_key(held[u]));
            } else {
                for (int i0 = tid; i0 < n; i0 += R * T) {
                    float x[R];
#pragma unroll
                    for (int u = 0; u < R; ++u) x[u] = i0 + u * T < n ? w[i0 + u * T] : 0.0f;
#pragma unroll
                    for (int u = 0; u < R; ++u)
                        if (i0 + u * T < n) f(value_key(x[u]));
                }
            }
        };
        uint32_t key = 0xffffffffu;  // the chosen lie over this key, and `left` at it
        if (left) {
            key = 0;
            for (int shift = 24; shift >= 0; shift -= 8) {
                for (int i = tid; i < COPIES * 256; i += T) sh.bins[i] = 0;
                if (tid == 0) sh.nfew = 0;
                __syncthreads();
                const uint32_t mask = shift == 24 ? 0u : ~0u << (shift + 8);
                each([&](uint32_t k) {
                    if ((k & mask) == key) atomicAdd(&sh.bins[lane % COPIES * 256 + (k >> shift & 255)], 1u);
                });
                __syncthreads();
                // A thread a bin: its count and how many lie over it.
                uint32_t mine = 0, upto = 0;
                if (tid < 256) {
#pragma unroll
                    for (int i = 0; i < COPIES; ++i) mine += sh.bins[i * 256 + tid];
                    upto = mine;
                    for (int d = 1; d < WAVE; d *= 2) {
                        const uint32_t x = __shfl_down(upto, d, WAVE);
                        if (lane + d < WAVE) upto += x;
                    }
                    if (lane == 0) sh.sums[wave] = upto;
                }
                __syncthreads();
                if (tid < 256) {
                    for (int i = wave + 1; i < 4; ++i) upto += sh.sums[i];
                    if (upto - mine < left && left <= upto)
                        sh.found[0] = uint32_t(tid), sh.found[1] = upto - mine, sh.found[2] = mine;
                }
                __syncthreads();
                key |= sh.found[0] << shift;
                left -= sh.found[1];
                if (shift && sh.found[2] <= FEW) {
                    const uint32_t m = sh.found[2], bits = ~0u << shift;
                    each([&](uint32_t k) {
                        if ((k & bits) == key) sh.few[atomicAdd(&sh.nfew, 1u)] = k;
                    });
                    __syncthreads();
                    if (uint32_t(tid) < m) {
                        uint32_t over = 0, upto = 0;
                        for (uint32_t j = 0; j < m; ++j) over += sh.few[j] > sh.few[tid], upto += sh.few[j] >= sh.few[tid];
                        if (over < left && left <= upto) sh.found[0] = sh.few[tid], sh.found[1] = over;
                    }
                    __syncthreads();
                    key = sh.found[0], left -= sh.found[1];
                    break;
                }
            }
        }
        // Values over the key and at it, by cells of 64.
        uint32_t over = 0, at = 0;  // before this part
        for (int base = 0; base < n; base += CELLS * WAVE) {
            const int end = n - base < CELLS * WAVE ? n - base : CELLS * WAVE;
            const int ncell = (end + WAVE - 1) / WAVE;
            auto count = [&](int c, int i, float x) {
                const uint32_t k = value_key(x);
                const uint64_t bo = __ballot(i < n && k > key), be = __ballot(i < n && k == key);
                if (lane == 0) sh.cells[2 * c] = __popcll(bo), sh.cells[2 * c + 1] = __popcll(be);
            };
            if constexpr (HELD) {
#pragma unroll
                for (int u = 0; u < R; ++u)
                    if (u * WAVES + wave < ncell) count(u * WAVES + wave, tid + u * T, held[u]);
            } else {
                for (int c = wave; c < ncell; c += WAVES) {
                    const int i = base + c * WAVE + lane;
                    count(c, i, i < n ? w[i] : 0.0f);
                }
            }
            __syncthreads();
            // Each thread a cell: the counts before it.
            const uint32_t o = tid < ncell ? sh.cells[2 * tid] : 0, e = tid < ncell ? sh.cells[2 * tid + 1] : 0;
            uint32_t po = o, pe = e;
            for (int d = 1; d < WAVE; d *= 2) {
                const uint32_t x = __shfl_up(po, d, WAVE), y = __shfl_up(pe, d, WAVE);
                if (lane >= d) po += x, pe += y;
            }
            if (lane == WAVE - 1) sh.sums[2 * wave] = po, sh.sums[2 * wave + 1] = pe;
            __syncthreads();
            uint32_t to = over, te = at;
            for (int i = 0; i < WAVES; ++i) {
                if (i < wave) po += sh.sums[2 * i], pe += sh.sums[2 * i + 1];
                to += sh.sums[2 * i], te += sh.sums[2 * i + 1];
            }
            if (tid < ncell) sh.cells[2 * tid] = over + po - o, sh.cells[2 * tid + 1] = at + pe - e;
            __syncthreads();
            // A chosen value's rank is the number of the chosen before it.
            for (int c0 = 0; c0 < ncell; c0 += R * WAVES) {
                float x[R];
                int rank[R];
#pragma unroll
                for (int u = 0; u < R; ++u) {
                    const int i = base + (c0 + u * WAVES + wave) * WAVE + lane;
                    if constexpr (HELD)
                        x[u] = held[u];
                    else
                        x[u] = i < n ? w[i] : 0.0f;
                }
#pragma unroll
                for (int u = 0; u < R; ++u) {
                    const int c = c0 + u * WAVES + wave;
                    const int i = base + c * WAVE + lane;
                    rank[u] = -1;
                    if (c >= ncell) continue;
                    const uint32_t k = value_key(x[u]);
                    const uint64_t before = (uint64_t(1) << lane) - 1;
                    const uint64_t bo = __ballot(i < n && k > key), be = __ballot(i < n && k == key);
                    const uint32_t no = sh.cells[2 * c] + __popcll(bo & before), ne = sh.cells[2 * c + 1] + __popcll(be & before);
                    if (i < n && (k > key || (k == key && ne < left))) rank[u] = no + (ne < left ? ne : left);
                }
                if constexpr (!HELD) __syncthreads();
#pragma unroll
                for (int u = 0; u < R; ++u)
                    if (rank[u] >= 0) hand(rank[u], base + (c0 + u * WAVES + wave) * WAVE + lane, x[u]);
            }
            over = to, at = te;
            __syncthreads();
        }
    }
};

}  // namespace omg
