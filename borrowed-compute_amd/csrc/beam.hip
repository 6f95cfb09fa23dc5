// A step of beam search over rows of scores on the device: of a search's beams x vocabulary
// continuations, whose scores are the beam's sum plus the token's log probability, the k best.
//
// Mathematics. log p_i = x_i - m - log L with m the row's largest score and L = sum e^(x_i - m). Within a
// row the order is the scores' own, so a row's k best tokens by score are all that the search can
// take from it; between rows the sums and log L decide, in 64 bits (two rows' continuations may lie nearer
// than an f32 tells apart). The terms of L and a lane's sum of them are f32: by at most
// 2^-17 they move all of a row's continuations alike; from lane to lane and part to part L is a tree and 64 bits.
//
// k_beam_scan: one pass over the scores, which keeps of a row the sum and the largest score of every group
// of 256, nothing else: a wave takes a part of a row alone, 1024 scores a step, the next step's on their
// way. k_beam_join: a search's workgroup looks at its rows' groups, 16384 at a time. Every group's largest
// is a continuation, so what does not reach the k'th of them is not among the k best: only the k groups
// that do (and their equals) are read again. Of their continuations, 16384 at a time, those that reach it too
// go into a pool with the best so far, and a key's rank in it is the number of better ones. The pool holds
// 4096: where more reach, whatever the scores (a mask's equal ones), a quarter as many are taken at a
// time. (Always a quarter: 70 us for 6 searches of 16 beams and their 64 best, 36 so. The candidates taken from
// each part as it is read, as k_logprobs has it, cost the scan twice its time at 16 best and 100 times
// at 64.)
//
// The scan is bound by its read: 128 rows of 128256 scores 12.5 us, 5.3 TB/s. The join is one chain of a
// workgroup a search: 11 us beside it, 9.5 for a search of 4 beams of 151936; 64 best take 10 us more
// than the best alone.
#include "common.hpp"
#include "internal.hpp"

#include <math.h>

#include <algorithm>
#include <type_traits>

namespace bchip {

namespace {

constexpr uint32_t BM_MOST = 64;               // beams of a search, and continuations asked for
constexpr uint32_t BM_WAVES = 4;               // of a workgroup
constexpr int BM_EACH = 16;                    // scores a lane and step
constexpr uint32_t BM_STEP = 64 * BM_EACH;
constexpr uint32_t BM_GROUPS = 4;              // of a step: group r holds its scores 256 j + 64 r + 0 .. 63, j < 4
constexpr uint32_t BM_PARTS = 128;             // most parts of a row
constexpr uint32_t BM_JOIN = 1024;             // threads of the join (256 took 4 us more: it is one chain)
constexpr int BM_KEYS = 4;                     // groups, or continuations, a thread of it holds at once
constexpr uint32_t BM_ROUND = BM_JOIN * BM_KEYS;

struct BmParams {
    const float* scores;
    const float* sums;
    float* best;
    uint32_t* beam;
    uint32_t* token;
    float* highs;    // [row][groups]: the largest score
    float2* states;  // [row][parts]: the largest score, the sum of e^(score - it)
    uint32_t rows, vocab, beams, k;
    uint32_t groups, parts, steps;  // groups and parts of a row, steps of a part
};

template <int N>
__device__ __forceinline__ float ror(float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x120 + N, 0xf, 0xf, false));
}
__device__ __forceinline__ float at_lane(float x, int i) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), i)); }
// Over sixteen lanes, and over a wave.
__device__ __forceinline__ float row_max(float x) {
    x = fmaxf(x, ror<8>(x));
    x = fmaxf(x, ror<4>(x));
    x = fmaxf(x, ror<2>(x));
    return fmaxf(x, ror<1>(x));
}
__device__ __forceinline__ float wave_max(float x) {
    x = row_max(x);
    return fmaxf(fmaxf(at_lane(x, 0), at_lane(x, 16)), fmaxf(at_lane(x, 32), at_lane(x, 48)));
}
__device__ __forceinline__ float wave_sum(float x) {
    x += ror<8>(x);
    x += ror<4>(x);
    x += ror<2>(x);
    x += ror<1>(x);
    return (at_lane(x, 0) + at_lane(x, 16)) + (at_lane(x, 32) + at_lane(x, 48));
}

struct __attribute__((packed, aligned(4))) Float4Any {  // rows of an odd vocabulary start anywhere
    float x, y, z, w;
};

__global__ __launch_bounds__(64 * BM_WAVES) void k_beam_scan(const BmParams p) {
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t id = blockIdx.x * BM_WAVES + wave, row = id / p.parts, part = id - row * p.parts;
    if (row >= p.rows) return;
    const float* s = p.scores + (size_t)row * p.vocab;
    float* highs = p.highs + (size_t)row * p.groups;
    const uint64_t from = (uint64_t)part * p.steps * BM_STEP;
    const uint32_t end = (uint32_t)min((uint64_t)p.vocab, from + (uint64_t)p.steps * BM_STEP);
    float m = -INFINITY, l = 0.0f;

    // Lane t's scores of a step: base + 256 j + 4 t + 0 .. 3.
    auto load = [&](float (&v)[BM_EACH], uint64_t base) {
#pragma unroll
        for (int j = 0; j < BM_EACH / 4; j++) {
            const Float4Any x = *(const Float4Any*)(s + base + 256 * j + 4 * lane);
            v[4 * j] = x.x, v[4 * j + 1] = x.y, v[4 * j + 2] = x.z, v[4 * j + 3] = x.w;
        }
    };
    float v[BM_EACH], next[BM_EACH];
    const uint32_t whole = (uint32_t)((end - from) / BM_STEP), all = (uint32_t)((end - from - 1) / BM_STEP) + 1;
    if (whole > 0) load(next, from);
    for (uint32_t step = 0; step < all; step++) {
        const uint64_t base = from + (uint64_t)step * BM_STEP;
        if (step < whole) {
#pragma unroll
            for (int e = 0; e < BM_EACH; e++) v[e] = next[e];
            load(next, from + (uint64_t)min(step + 1, whole - 1) * BM_STEP);  // (no branch around it; the last one's again)
        } else {
#pragma unroll
            for (int e = 0; e < BM_EACH; e++) {
                const uint64_t i = base + 256 * (e >> 2) + 4 * lane + (e & 3);
                v[e] = i < end ? s[i] : -INFINITY;
            }
#pragma unroll
            for (int e = 0; e < BM_EACH; e++) asm volatile("" : "+v"(v[e]));  // (waited for here, not where the other way's next step would be)
        }
        float high = -INFINITY;
#pragma unroll
        for (int e = 0; e < BM_EACH; e++) high = fmaxf(high, v[e]);
        if (high > m) {
            l *= exp2_hw((m - high) * LOG2E);
            m = high;
        }
        const float ms = m == -INFINITY ? 0.0f : m;
        float sum = 0.0f;
#pragma unroll
        for (int e = 0; e < BM_EACH; e++) sum += exp2_hw((v[e] - ms) * LOG2E);
        l += sum;
        high = row_max(high);
        if ((lane & 15) == 0) highs[(base / BM_STEP) * BM_GROUPS + lane / 16] = high;
    }
    const float M = wave_max(m);
    l = wave_sum(m == -INFINITY ? l : l * exp2_hw((m - M) * LOG2E));
    if (lane == 0) p.states[id] = float2{M, l};
}

struct BmKey {
    uint64_t score;  // ascending with the score; 0: none, 1: not a number
    uint64_t place;  // beam << 32 | token
    __device__ __forceinline__ bool above(const BmKey& o) const { return score != o.score ? score > o.score : place < o.place; }
};
__device__ __forceinline__ uint64_t bm_order(double v) {
    const uint64_t bits = __double_as_longlong(v);
    return v != v ? 1 : bits >> 63 ? ~bits : bits | 1ull << 63;
}

// The k'th largest of the threads' numbers, of every four the largest, by their upper halves (the smallest
// that fewer than k are larger than: k of them reach it). Every thread calls it; least: LDS, ~0 before.
__device__ __forceinline__ uint64_t bm_reach(uint64_t top, uint32_t k, uint32_t* highs, uint32_t* least) {
    uint32_t high = (uint32_t)(top >> 32);
    high = max(high, (uint32_t)__shfl_xor((int)high, 1));
    high = max(high, (uint32_t)__shfl_xor((int)high, 2));
    if ((threadIdx.x & 3) == 0) highs[threadIdx.x / 4] = high;
    __syncthreads();
    uint32_t larger = 0;  // (a quarter of them each, for the four's largest)
#pragma unroll 8
    for (uint32_t i = 0; i < BM_JOIN / 16; i += 4) {
        const uint4 x = *(const uint4*)&highs[4 * i + 4 * (threadIdx.x & 3)];
        larger += (uint32_t)(x.x > high) + (uint32_t)(x.y > high) + (uint32_t)(x.z > high) + (uint32_t)(x.w > high);
    }
    larger += (uint32_t)__shfl_xor((int)larger, 1);
    larger += (uint32_t)__shfl_xor((int)larger, 2);
    uint32_t low = larger < k ? high : ~0u;
#pragma unroll
    for (int d = 4; d < 64; d *= 2) low = min(low, (uint32_t)__shfl_xor((int)low, d));
    if ((threadIdx.x & 63) == 0) atomicMin(least, low);
    __syncthreads();
    return (uint64_t)*least << 32;
}

__global__ __launch_bounds__(BM_JOIN) void k_beam_join(const BmParams p) {
    __shared__ double base[BM_MOST];  // a beam's sum less its row's largest score and log L
    __shared__ BmKey pool[BM_ROUND + BM_MOST], best[BM_MOST];
    __shared__ uint64_t floor;
    __shared__ __attribute__((aligned(16))) uint32_t list[BM_ROUND], highs[BM_JOIN / 4], least, listed, count;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const size_t row0 = (size_t)blockIdx.x * p.beams;
    const uint32_t all = p.beams * p.groups;
    constexpr int WIDE = 4 * BM_KEYS;
    float high[WIDE];
    auto load = [&](uint32_t g0, bool wide) {  // (no branch around either's loads: all on their way at once)
#pragma unroll
        for (int i = 0; i < BM_KEYS; i++) high[i] = p.highs[row0 * p.groups + min(g0 + BM_JOIN * i + tid, all - 1)];
        if (wide)
#pragma unroll
            for (int i = BM_KEYS; i < WIDE; i++) high[i] = p.highs[row0 * p.groups + min(g0 + BM_JOIN * i + tid, all - 1)];
    };
    load(0, all > BM_ROUND);
    for (uint32_t b = wave; b < p.beams; b += BM_JOIN / 64) {
        const float2* states = p.states + (row0 + b) * p.parts;
        const float2 none = {-INFINITY, 0.0f}, x = lane < p.parts ? states[lane] : none, y = lane + 64 < p.parts ? states[lane + 64] : none;
        const float M = wave_max(fmaxf(x.x, y.x));
        // (A part of nothing but -inf has a sum of 0, one with a NaN a NaN.)
        double l = (x.x == -INFINITY ? (double)x.y : (double)x.y * exp((double)x.x - (double)M)) +
                   (y.x == -INFINITY ? (double)y.y : (double)y.y * exp((double)y.x - (double)M));
#pragma unroll
        for (int d = 1; d < 64; d *= 2) l += __shfl_xor(l, d);
        if (lane == 0) base[b] = (double)p.sums[row0 + b] - ((double)M + log(l));
    }
    if (tid == 0) {
        listed = count = 0;
        least = ~0u;
        floor = ~0ull;
    }
    uint32_t kept = 0;
    const float per = 1.0f / p.groups;
    __syncthreads();
    // Groups from g0 on, N a thread: those that reach the k'th largest of the threads' go into the pool, those of
    // them that fewer than k are larger than on the list. False where the pool has no room for all.
    auto look = [&](uint32_t g0, auto each) {
        constexpr int N = decltype(each)::value;
        uint64_t order[N], top = 0;
        uint32_t place[N], more = 0;
#pragma unroll
        for (int i = 0; i < N; i++) {
            const uint32_t g = min(g0 + BM_JOIN * i + tid, all - 1);
            uint32_t b = (uint32_t)((float)g * per);  // g / p.groups, or one beside it
            b -= b * p.groups > g;
            b += (b + 1) * p.groups <= g;
            // (A row's last groups may lie past its end, and are none of it: their -inf would stand above a NaN.)
            const uint32_t in = g - b * p.groups, first = in / BM_GROUPS * BM_STEP + 64 * (in % BM_GROUPS);
            order[i] = g0 + BM_JOIN * i + tid < all && first < p.vocab ? bm_order(base[b] + (double)high[i]) : 0;
            place[i] = b << 25 | in;
            top = top > order[i] ? top : order[i];
        }
        const uint64_t reach = bm_reach(top, p.k, highs, &least), worst = kept == p.k ? best[p.k - 1].score : 0, from = reach > worst ? reach : worst;
#pragma unroll
        for (int i = 0; i < N; i++) {
            if (order[i] < from) order[i] = 0;
            more += order[i] != 0;
        }
        if (N > BM_KEYS && __syncthreads_count(more > BM_KEYS)) {
            if (tid == 0) least = ~0u;
            __syncthreads();
            return false;
        }
#pragma unroll
        for (int i = 0; i < N; i++)
            if (order[i] != 0) pool[atomicAdd(&count, 1u)] = BmKey{order[i], place[i]};
        __syncthreads();
        const uint32_t n = count;
        for (uint32_t i = tid; i < n; i += BM_JOIN) {
            const uint64_t x = pool[i].score;
            uint32_t larger = 0;
#pragma unroll 8
            for (uint32_t j = 0; j < n; j++) larger += pool[j].score > x;
            if (larger < p.k) {
                list[atomicAdd(&listed, 1u)] = (uint32_t)pool[i].place;
                atomicMin((unsigned long long*)&floor, (unsigned long long)x);
            }
        }
        __syncthreads();
        return true;
    };
    uint32_t narrow = 0;  // rounds of BM_ROUND to come in place of one of four times as many
    for (uint32_t g0 = 0; g0 < all;) {
        const bool wide = narrow == 0 && all - g0 > BM_ROUND;
        if (g0 > 0) load(g0, wide);
        if (wide) {
            if (!look(g0, std::integral_constant<int, WIDE>())) {
                narrow = WIDE / BM_KEYS;
                continue;
            }
        } else {
            look(g0, std::integral_constant<int, BM_KEYS>());
            narrow -= narrow > 0;
        }
        g0 += wide ? WIDE * BM_JOIN : BM_ROUND;
        const uint32_t found = listed;
        if (tid == 0) {
            count = 0;
            least = ~0u;
        }
        // Their continuations, those of 4 N groups from l0 on: N a thread. What reaches the k'th of the groups (with
        // fewer of them nothing is known of the k'th continuation) and the best so far goes into the pool; of
        // many (good tokens that lie side by side) what reaches the k'th largest of the threads'. False where
        // the pool has no room for all.
        auto take = [&](uint32_t l0, auto each) {
            constexpr int N = decltype(each)::value;
            const uint64_t from = found >= p.k ? floor : 0;
            float v[N];
            auto of = [&](int i, uint32_t& b) {  // the token
                const uint32_t x = list[min(l0 + BM_JOIN / 256 * i + tid / 256, found - 1)], in = x & 0x1ffffffu;
                b = x >> 25;
                return (uint64_t)(in / BM_GROUPS) * BM_STEP + 256 * (wave & 3) + 64 * (in % BM_GROUPS) + lane;
            };
#pragma unroll
            for (int i = 0; i < N; i++) {
                uint32_t b;
                const uint64_t t = of(i, b);
                v[i] = p.scores[(row0 + b) * p.vocab + (t < p.vocab ? t : p.vocab - 1)];
            }
            __syncthreads();  // (count)
            BmKey mine[N];
            const BmKey last = best[p.k - 1];
            uint64_t top = 0;
            uint32_t more = 0;
#pragma unroll
            for (int i = 0; i < N; i++) {
                uint32_t b;
                const uint64_t t = of(i, b);
                mine[i] = BmKey{l0 + BM_JOIN / 256 * i + tid / 256 < found && t < p.vocab ? bm_order(base[b] + (double)v[i]) : 0, (uint64_t)b << 32 | t};
                if (mine[i].score < from || (kept == p.k && !mine[i].above(last))) mine[i].score = 0;
                top = top > mine[i].score ? top : mine[i].score;
                more += mine[i].score != 0;
            }
            if (__syncthreads_count(more > 2)) {
                const uint64_t reach = bm_reach(top, p.k, highs, &least);
                more = 0;
#pragma unroll
                for (int i = 0; i < N; i++) {
                    if (mine[i].score < reach) mine[i].score = 0;
                    more += mine[i].score != 0;
                }
                if (N > BM_KEYS && __syncthreads_count(more > BM_KEYS)) {
                    if (tid == 0) least = ~0u;
                    __syncthreads();
                    return false;
                }
            }
#pragma unroll
            for (int i = 0; i < N; i++)
                if (mine[i].score != 0) pool[atomicAdd(&count, 1u)] = mine[i];
            __syncthreads();
            if (tid < kept) pool[count + tid] = best[tid];
            __syncthreads();
            const uint32_t n = count + kept;
            for (uint32_t i = tid; i < n; i += BM_JOIN) {
                const BmKey x = pool[i];
                uint32_t rank = 0;
#pragma unroll 8
                for (uint32_t j = 0; j < n; j++) rank += pool[j].above(x);
                if (rank < p.k) best[rank] = x;
            }
            __syncthreads();
            if (tid == 0) {
                count = 0;
                least = ~0u;
            }
            kept = min(n, p.k);
            return true;
        };
        constexpr uint32_t ROUND = BM_ROUND / 256;  // groups
        if (found <= 2 * ROUND || found > 4 * ROUND || !take(0, std::integral_constant<int, WIDE>()))
            for (uint32_t l0 = 0; l0 < found; l0 += ROUND) take(l0, std::integral_constant<int, BM_KEYS>());
        __syncthreads();
        if (tid == 0) {
            listed = count = 0;
            least = ~0u;
            floor = ~0ull;
        }
        __syncthreads();
    }
    if (tid < p.k) {
        const BmKey x = best[tid];
        const uint64_t bits = x.score >> 63 ? x.score & ~(1ull << 63) : ~x.score;
        const size_t at = (size_t)blockIdx.x * p.k + tid;
        p.best[at] = x.score == 1 ? NAN : (float)__longlong_as_double(bits);
        p.beam[at] = (uint32_t)(x.place >> 32);
        p.token[at] = (uint32_t)x.place;
    }
}

// Parts of a row: as many as keep every SIMD at four waves, where a row has the steps.
void plan(BmParams& p) {
    const uint32_t steps = (p.vocab - 1) / BM_STEP + 1;
    const uint32_t parts = std::min(std::max(1u, 4096u / p.rows), std::min(steps, BM_PARTS));
    p.steps = (steps + parts - 1) / parts;
    p.parts = (steps + p.steps - 1) / p.steps;
    p.groups = steps * BM_GROUPS;
}

}  // namespace

size_t beam_scratch_bytes(uint32_t rows, uint32_t vocab) {
    BmParams p{};
    p.rows = rows;
    p.vocab = vocab;
    plan(p);
    return (size_t)rows * (p.groups * sizeof(float) + p.parts * sizeof(float2));
}

hipError_t beam_launch(const float* scores, const float* sums, uint32_t batch, uint32_t beams, uint32_t vocab, uint32_t k,
                       float* best, uint32_t* beam, uint32_t* token, void* scratch, hipStream_t s) {
    BmParams p{scores, sums, best, beam, token, (float*)scratch, nullptr, batch * beams, vocab, beams, k, 0, 0, 0};
    plan(p);
    p.states = (float2*)(p.highs + (size_t)p.rows * p.groups);  // (groups are fours)
    hipLaunchKernelGGL(k_beam_scan, dim3((uint32_t)(((uint64_t)p.rows * p.parts + BM_WAVES - 1) / BM_WAVES)), dim3(64 * BM_WAVES), 0, s, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(k_beam_join, dim3(batch), dim3(BM_JOIN), 0, s, p);
    return hipGetLastError();
}

}  // namespace bchip
