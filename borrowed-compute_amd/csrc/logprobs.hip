// Log probabilities of given tokens, the entropy of their distribution and the most likely
// tokens, from rows of scores on the device: what the step beside the sampler (sample.hip) says
// about a choice instead of making it.
//
// Mathematics, per row: m = the largest score, x_i = (s_i - m) / T, L = sum e^x_i, A = sum e^x_i
// x_i. Then log p_i = x_i - log L and the entropy is log L - A / L. L is kept as c, the terms that
// are 1, and L1, the sum of the others: where one token holds nearly everything log L =
// log1p(L1) keeps its digits. States of parts of a row, each against its own m, meet by
// L -> e^d L, A -> e^d (A + d L) with d = (m' - m) / T.
//
// One pass over the scores. A workgroup holds a block of 8192 in registers (32 a thread) and takes
// from it the sums and the candidates for the best tokens. A row's first block has none to compare
// with: of the maxima of 64 groups of threads, or of all 256 threads, the top'th largest has `top`
// scores at or above it. Later blocks leave what is above the worst number kept, few or none. A wave
// puts its candidates into LDS by the counts of its ballots, and a key's rank is the number of
// better ones. Blocks whose candidates are too many (most scores equal, as under a mask) pick the
// best one at a time. Keys of score over inverted index make every order total: ties go to the
// lowest index, a NaN is behind every number.
//
// A row's sums are kept by units (a block, or several where a row has more than 64) and meet in one
// order, so its bits do not depend on how many workgroups share it: as many as make 2048 a launch;
// k_logprobs_join brings a row's together.
//
// Measured, scores in f32, with the join: 1 row of 151936 7.0 us without best tokens and 11.7 with 5,
// latency; 256 rows of 128256 27.9 us without (4.7 TB/s), 46 with 20, 62 with 64; 1024 rows 95.6
// (5.5 TB/s, what reading alone reaches) and 137 with 20, where the selection's registers leave three
// workgroups a CU instead of eight. Blocks of 4096 take 28 us for one row with 20 and the same time
// for many; 768 workgroups 159 us for those 1024 rows, whose last round is a third full.
#include "common.hpp"
#include "internal.hpp"

#include <math.h>

#include <algorithm>

namespace bchip {

namespace {

constexpr int LP_THREADS = 256, LP_EACH = 32;
constexpr uint32_t LP_BLOCK = LP_THREADS * LP_EACH;  // scores a workgroup holds at once
constexpr uint32_t LP_TOP = 64;                      // most tokens a row is asked for
constexpr uint32_t LP_SEG = 160;                     // candidates of a wave
constexpr uint32_t LP_RANK = 64;                     // as many of a wave are ranked
constexpr uint32_t LP_PARTS = 64;                    // most units of a row, and workgroups
constexpr uint32_t LP_GROUPS = 2048;                 // workgroups of a launch, where rows have the blocks

// Ascending keys are ascending scores, lower indices first among equals read downwards; 0 is no
// token at all, and a NaN comes next.
__device__ __forceinline__ uint64_t lp_key(float s, uint32_t i) {
    const uint32_t b = __float_as_uint(s + 0.0f);  // (-0 is 0)
    const uint32_t o = s != s ? 1u : (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    return (uint64_t)o << 32 | (0xffffffffu - i);
}
__device__ __forceinline__ float lp_score(uint64_t key) {
    const uint32_t o = (uint32_t)(key >> 32);
    return o == 1u ? NAN : __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}
__device__ __forceinline__ uint32_t lp_index(uint64_t key) { return 0xffffffffu - (uint32_t)key; }

struct LpState {
    float m, c, l, a;
};

// A state against its own m to one against M >= m.
__device__ __forceinline__ void lp_rebase(LpState& s, float M, float k) {
    if (s.m == M) return;
    const float d = fmaxf((s.m - M) * k, -1e4f), x = exp2_hw(d), l = s.c + s.l;
    s.a = x * (s.a + d * l);
    s.l = x * l;
    s.c = 0.0f;
    s.m = M;
}

struct LpParams {
    const float* scores;
    const uint32_t* tokens;
    float* logprob;
    float* entropy;
    uint32_t* ids;
    float* tops;
    LpState* states;  // [row][units]
    uint64_t* keys;   // [row][parts][top]
    uint32_t vocab, top;
    uint32_t units, blocks;  // units of a row, blocks of LP_BLOCK scores a unit
    uint32_t parts, per;     // workgroups of a row, units a workgroup
    float inv_t, k;  // 1 / T, log2 e / T
};

// What a row's whole state and its best keys (in LDS, best first) say.
__device__ __forceinline__ void lp_finish(const LpParams& p, uint32_t row, const LpState& s, const uint64_t* best) {
    const uint32_t tid = threadIdx.x;
    const float log_l = s.c == 1.0f ? log1pf(s.l) : logf(s.c + s.l);
    if (tid == 0) {
        if (p.logprob) {
            const uint32_t t = p.tokens[row];
            p.logprob[row] = t < p.vocab ? (p.scores[(size_t)row * p.vocab + t] - s.m) * p.inv_t - log_l : NAN;
        }
        if (p.entropy) p.entropy[row] = log_l - 0.69314718f * s.a / (s.c + s.l);
    }
    if (tid < p.top) {
        const uint64_t k = best[tid];
        p.ids[(size_t)row * p.top + tid] = lp_index(k);
        p.tops[(size_t)row * p.top + tid] = (lp_score(k) - s.m) * p.inv_t - log_l;
    }
}

// Keys of pool[0 .. n) above k; zeros follow up to a multiple of eight.
__device__ __forceinline__ uint32_t lp_above(const uint64_t* pool, uint32_t n, uint64_t k) {
    uint32_t above = 0;
    for (uint32_t j = 0; j < n; j += 8)  // (the reads of eight do not wait for each other)
#pragma unroll
        for (int e = 0; e < 8; e++) above += pool[j + e] > k;
    return above;
}

// The least float above x.
__device__ __forceinline__ float next_up(float x) {
    const uint32_t b = __float_as_uint(x);
    return __uint_as_float(x == 0.0f ? 1u : x > 0.0f ? b + 1 : b - 1);
}

// Over a wave: rotations within 16 lanes, then the four sixteens' values by name.
template <int N>
__device__ __forceinline__ float ror(float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x120 + N, 0xf, 0xf, false));
}
__device__ __forceinline__ float at_lane(float x, int i) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), i)); }
__device__ __forceinline__ float wave_max(float x) {
    x = fmaxf(x, ror<8>(x));
    x = fmaxf(x, ror<4>(x));
    x = fmaxf(x, ror<2>(x));
    x = fmaxf(x, ror<1>(x));
    return fmaxf(fmaxf(at_lane(x, 0), at_lane(x, 16)), fmaxf(at_lane(x, 32), at_lane(x, 48)));
}
__device__ __forceinline__ float wave_sum(float x) {
    x += ror<8>(x);
    x += ror<4>(x);
    x += ror<2>(x);
    x += ror<1>(x);
    return (at_lane(x, 0) + at_lane(x, 16)) + (at_lane(x, 32) + at_lane(x, 48));
}

// A row's state from its units', one a lane.
__device__ __forceinline__ LpState lp_row(LpState s, float k) {
    lp_rebase(s, wave_max(s.m), k);
    s.c = wave_sum(s.c);
    s.l = wave_sum(s.l);
    s.a = wave_sum(s.a);
    return s;
}

struct __attribute__((packed, aligned(4))) Float4Any {  // rows of an odd vocabulary start anywhere
    float x, y, z, w;
};

template <bool TOP>
__global__ __launch_bounds__(LP_THREADS, TOP ? 3 : 8) void k_logprobs(const LpParams p) {
    __shared__ uint64_t cand[4][TOP ? LP_SEG : 1], best[2][TOP ? LP_TOP : 1], pick[4];
    __shared__ LpState waves[LP_PARTS][4], whole;
    __shared__ float red[4];
    __shared__ __attribute__((aligned(16))) float gmax[TOP ? LP_THREADS : 1];
    __shared__ uint32_t cnt[2][4];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), row = blockIdx.y, part = blockIdx.x;
    const float* s = p.scores + (size_t)row * p.vocab;
    LpState st{-INFINITY, 0.0f, 0.0f, 0.0f};
    const uint32_t u0 = part * p.per, nu = min(p.per, p.units - u0);
    uint32_t which = 0, kept = 0;          // best[which] holds `kept` keys, in order,
    uint32_t mine = 0, c[4] = {}, n = 0;   // cand the candidates since, a wave's and every wave's; n of all
    bool full = false, over = false;       // best holds `top` numbers,
    float floor = -INFINITY;               // of which this is the smallest
    uint32_t flip = 0;
    if (TOP && tid < 2 * LP_TOP) best[tid / LP_TOP][tid % LP_TOP] = 0;  // (waited for before any rank)
    for (uint32_t b = 0, u = 0, next = p.blocks; u < nu; b++) {
        const uint64_t base = ((uint64_t)u0 * p.blocks + b) * LP_BLOCK;
        const bool end = base + LP_BLOCK >= p.vocab;
        // Thread t's scores: base + 1024 j + 4 t + 0 .. 3.
        float v[LP_EACH];
        auto index = [&](int e) { return (uint32_t)base + 4u * LP_THREADS * (e >> 2) + 4u * tid + (e & 3); };
#pragma unroll
        for (int j = 0; j < LP_EACH / 4; j++) {
            const uint64_t i = base + 4u * LP_THREADS * j + 4u * tid;
            if (i + 4 <= p.vocab) {
                const Float4Any x = *(const Float4Any*)(s + i);
                v[4 * j] = x.x, v[4 * j + 1] = x.y, v[4 * j + 2] = x.z, v[4 * j + 3] = x.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) v[4 * j + e] = i + e < p.vocab ? s[i + e] : -INFINITY;
            }
        }
        float top = -INFINITY;
#pragma unroll
        for (int e = 0; e < LP_EACH; e++) top = fmaxf(top, v[e]);
        lp_rebase(st, fmaxf(st.m, top), p.k);
        const float m = st.m == -INFINITY ? 0.0f : st.m;
        uint32_t ones = 0;
#pragma unroll
        for (int e = 0; e < LP_EACH; e++) {
            const float x = (v[e] - m) * p.k, w = exp2_hw(x);
            st.l += x == 0.0f ? 0.0f : w;
            ones += x == 0.0f;
            st.a = __builtin_fmaf(w, fmaxf(x, -1e4f), st.a);  // (0 for a score of -inf; a NaN stays one)
        }
        st.c += (float)ones;
        if (b + 1 == next || end) {  // of the unit
            lp_rebase(st, wave_max(st.m), p.k);
            st.c = wave_sum(st.c);
            st.l = wave_sum(st.l);
            st.a = wave_sum(st.a);
            if (lane == 0) waves[u][wave] = st;
            st = LpState{-INFINITY, 0.0f, 0.0f, 0.0f};
            next += p.blocks;
            u++;
        }
        if constexpr (!TOP) continue;
        // Candidates are the scores above the worst number kept, which beats its equals of later
        // blocks. Without as many numbers as asked for, or where too many are above it: those that reach
        // the top'th largest of the block's groups' maxima, which at least `top` of its scores do, and of
        // them those above -inf (under a mask those alone, if they are enough).
        const uint32_t had = mine, hads = n, here = (uint32_t)min((uint64_t)LP_BLOCK, p.vocab - base);
        auto tell = [&]() {  // each wave's candidates, zeros behind them up to eights
            if (lane < 8 && mine + lane < LP_SEG) cand[wave][mine + lane] = 0;
            if (lane == 0) cnt[flip][wave] = mine;
            __syncthreads();
            n = kept;
            over = false;
#pragma unroll
            for (int w = 0; w < 4; w++) {
                c[w] = __builtin_amdgcn_readfirstlane(cnt[flip][w]);
                n += c[w];
                over |= c[w] > LP_SEG;
            }
            flip ^= 1;
        };
        for (bool all = full;; all = false) {
            float least = next_up(floor);
            if (!all) {
                const uint32_t groups = p.top <= 32 ? 64 : LP_THREADS;
                float gm = top;
                if (groups == 64) {  // four threads a group
                    gm = fmaxf(gm, __shfl_xor(gm, 1));
                    gm = fmaxf(gm, __shfl_xor(gm, 2));
                }
                if (groups == LP_THREADS) gmax[tid] = gm;
                else if ((tid & 3) == 0) gmax[tid >> 2] = gm;
                __syncthreads();
                // The smallest of those that fewer than `top` are larger than; a wave looks at 64 of them.
                const float at = gmax[(groups == 64 ? 0 : 64 * wave) + lane];
                uint32_t above = 0;
                for (uint32_t j = 0; j < groups; j += 16)
#pragma unroll
                    for (int e = 0; e < 16; e += 4) {
                        const float4 x = *(const float4*)&gmax[j + e];
                        above += (uint32_t)(x.x > at) + (uint32_t)(x.y > at) + (uint32_t)(x.z > at) + (uint32_t)(x.w > at);
                    }
                float low = -wave_max(above < p.top ? -at : -INFINITY);
                if (groups != 64) {
                    if (lane == 0) red[wave] = low;
                    __syncthreads();
                    low = fminf(fminf(red[0], red[1]), fminf(red[2], red[3]));
                }
                least = fmaxf(least, low);
            }
            mine = had;
            if (__any(top >= least)) {
#pragma unroll
                for (int e = 0; e < LP_EACH; e++) {
                    const bool is = v[e] >= least;
                    const uint64_t them = __ballot(is);
                    if (them) {
                        const uint32_t at = mine + __builtin_amdgcn_mbcnt_hi((uint32_t)(them >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)them, 0));
                        if (is && at < LP_SEG) cand[wave][at] = lp_key(v[e], index(e));
                        mine += __popcll(them);
                    }
                }
            }
            tell();
            if (!all || !over) break;
        }
        // Candidates that are fewer than asked for may leave out scores of -inf and NaNs.
        const bool few = !full && (n < p.top || kept == p.top) && n - hads < here;
        if (few || over) {
            uint32_t taken = 0;
            mine = had;
            for (uint32_t r = 0; r < min(p.top, here); r++) {
                uint64_t k = 0;
#pragma unroll
                for (int e = 0; e < LP_EACH; e++)
                    if (!(taken >> e & 1u) && index(e) - (uint32_t)base < here) k = max(k, lp_key(v[e], index(e)));
                uint64_t w = k;
#pragma unroll
                for (int d = 1; d < 64; d *= 2) w = max(w, (uint64_t)__shfl_xor((unsigned long long)w, d));
                if (lane == 0) pick[wave] = w;
                __syncthreads();
                const uint64_t x = max(max(pick[0], pick[1]), max(pick[2], pick[3]));
                __syncthreads();
                if (x == k) {  // (keys are unique: one thread's)
                    const uint32_t off = lp_index(k) - (uint32_t)base;
                    taken |= 1u << (off / (4 * LP_THREADS) * 4 + (off & 3));
                    cand[wave][mine] = k;
                }
                if (x == w) mine++;
            }
            tell();
        }
        // Ranked where there were too few numbers, where many have come together, and at the end.
        const bool last = u == nu;
        if (!full || last || max(max(c[0], c[1]), max(c[2], c[3])) > LP_RANK) {
            uint64_t* to = best[which ^ 1];
            for (uint32_t i = tid; i < n; i += LP_THREADS) {
                uint32_t x = i;
                const uint64_t* at = best[which];
                if (x >= kept) {
                    x -= kept;
                    int w = 0;
                    for (; w < 3 && x >= c[w]; w++) x -= c[w];
                    at = cand[w];
                }
                const uint64_t k = at[x];
                uint32_t rank = lp_above(best[which], kept, k);
#pragma unroll
                for (int w = 0; w < 4; w++) rank += lp_above(cand[w], c[w], k);
                if (rank < p.top) to[rank] = k;
            }
            __syncthreads();
            which ^= 1;
            kept = n = min(n, p.top);
            mine = 0;
            const float worst = kept == p.top ? lp_score(to[p.top - 1]) : NAN;
            full = worst == worst;
            floor = full ? worst : -INFINITY;
        }
    }
    __syncthreads();
    if (tid < 64) {
        LpState x{-INFINITY, 0.0f, 0.0f, 0.0f};
        if (tid < nu) {
            const float M = fmaxf(fmaxf(waves[tid][0].m, waves[tid][1].m), fmaxf(waves[tid][2].m, waves[tid][3].m));
            x.m = M;
            for (int w = 0; w < 4; w++) {
                LpState y = waves[tid][w];
                lp_rebase(y, M, p.k);
                x.c += y.c;
                x.l += y.l;
                x.a += y.a;
            }
            if (p.parts > 1) p.states[(size_t)row * p.units + u0 + tid] = x;
        }
        if (p.parts == 1) {
            x = lp_row(x, p.k);
            if (tid == 0) whole = x;
        }
    }
    if (p.parts == 1) {
        __syncthreads();
        lp_finish(p, row, whole, best[which]);
        return;
    }
    if (TOP && tid < p.top) p.keys[((size_t)row * p.parts + part) * p.top + tid] = tid < kept ? best[which][tid] : 0;
}

template <bool TOP>
__global__ __launch_bounds__(LP_THREADS) void k_logprobs_join(const LpParams p) {
    constexpr int MOST = LP_PARTS * LP_TOP / LP_THREADS;  // keys a thread
    __shared__ uint64_t pool[TOP ? LP_PARTS * LP_TOP + 8 : 1], best[TOP ? LP_TOP : 1];
    __shared__ uint64_t low[LP_PARTS];
    __shared__ LpState all;
    __shared__ uint32_t count;
    const uint32_t tid = threadIdx.x, row = blockIdx.x;
    const LpState* states = p.states + (size_t)row * p.units;
    uint64_t k[TOP ? MOST : 1];
    // Every part's keys are in order: with ceil(top / parts) of each at or above the smallest
    // of those, `top` are.
    const uint32_t keys = p.parts * p.top, each = (p.top + p.parts - 1) / p.parts;
    if constexpr (TOP) {
#pragma unroll
        for (int i = 0; i < MOST; i++) {
            const uint32_t x = tid + i * LP_THREADS;
            if (i * LP_THREADS < keys) {
                k[i] = x < keys ? p.keys[(size_t)row * keys + x] : 0;
                if (x < keys && x % p.top == each - 1) low[x / p.top] = k[i];
            }
        }
    }
    if (tid < 64) {  // LP_PARTS is a wave
        const LpState s = lp_row(tid < p.units ? states[tid] : LpState{-INFINITY, 0.0f, 0.0f, 0.0f}, p.k);
        if (tid == 0) {
            all = s;
            count = 0;
        }
    }
    __syncthreads();
    if constexpr (TOP) {
        uint64_t least = low[0];
#pragma unroll 8
        for (uint32_t i = 1; i < p.parts; i++) least = min(least, low[i]);
#pragma unroll
        for (int i = 0; i < MOST; i++)
            if (i * LP_THREADS < keys && k[i] >= least && k[i] != 0) pool[atomicAdd(&count, 1u)] = k[i];
        __syncthreads();
        const uint32_t n = count;
        if (tid < 8) pool[n + tid] = 0;
        __syncthreads();
        for (uint32_t i = tid; i < n; i += LP_THREADS) {
            const uint64_t x = pool[i];
            const uint32_t rank = lp_above(pool, n, x);
            if (rank < p.top) best[rank] = x;
        }
        __syncthreads();
    }
    lp_finish(p, row, all, best);
}

// Blocks a unit, units a row, and units a workgroup of `rows` rows.
void lp_plan(uint32_t rows, uint32_t vocab, LpParams& p) {
    const uint32_t all = (vocab - 1) / LP_BLOCK + 1;
    p.blocks = (all + LP_PARTS - 1) / LP_PARTS;
    p.units = (all + p.blocks - 1) / p.blocks;
    p.per = (p.units + (LP_GROUPS + rows - 1) / rows - 1) / ((LP_GROUPS + rows - 1) / rows);
    p.parts = (p.units + p.per - 1) / p.per;
}

}  // namespace

// At most 4.2 MB: parts times rows is below 2 LP_GROUPS, and from LP_GROUPS rows on a row has one
// workgroup and the call no scratch.
size_t logprobs_scratch_bytes(uint32_t rows, uint32_t vocab, uint32_t top) {
    LpParams p{};
    lp_plan(rows, vocab, p);
    return p.parts == 1 ? 0 : (size_t)rows * (p.units * sizeof(LpState) + (size_t)p.parts * top * sizeof(uint64_t));
}

hipError_t logprobs_launch(const float* scores, uint32_t rows, uint32_t vocab, float temperature, const uint32_t* tokens,
                           float* logprob, float* entropy, uint32_t top, uint32_t* ids, float* tops, void* scratch,
                           hipStream_t s) {
    LpParams p{};
    p.scores = scores;
    p.tokens = tokens;
    p.logprob = logprob;
    p.entropy = entropy;
    p.ids = ids;
    p.tops = tops;
    p.vocab = vocab;
    p.top = top;
    lp_plan(rows, vocab, p);
    if (!scratch) {
        p.parts = 1;
        p.per = p.units;
    }
    p.inv_t = 1.0f / temperature;
    p.k = (float)(1.4426950408889634 / (double)temperature);
    p.keys = (uint64_t*)scratch;
    p.states = (LpState*)((uint64_t*)scratch + (size_t)rows * p.parts * top);
    hipLaunchKernelGGL(top ? k_logprobs<true> : k_logprobs<false>, dim3(p.parts, rows), dim3(LP_THREADS), 0, s, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.parts == 1) return e;
    hipLaunchKernelGGL(top ? k_logprobs_join<true> : k_logprobs_join<false>, dim3(rows), dim3(LP_THREADS), 0, s, p);
    return hipGetLastError();
}

}  // namespace bchip
