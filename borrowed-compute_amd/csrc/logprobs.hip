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
// One pass over the scores. A workgroup holds 8192 of them in registers (32 a thread) and takes
// from them their maximum, the sums and the block's best tokens: of the maxima of 64 groups of
// threads, or of all 256 threads, the top'th largest has `top` scores at or above it, so only
// those, little more than `top`, go into LDS, where each one's rank is the number of better ones.
// Rows whose candidates are too many (most scores equal, as under a mask) pick the block's best one
// at a time. Keys of score over inverted index make every order total: ties go to the lowest
// index, a NaN is behind every number. Rows are cut over workgroups; k_logprobs_join brings a
// row's parts together.
#include "common.hpp"
#include "internal.hpp"

#include <math.h>

#include <algorithm>

namespace bchip {

namespace {

constexpr int LP_THREADS = 256, LP_EACH = 32;
constexpr uint32_t LP_BLOCK = LP_THREADS * LP_EACH;  // scores a workgroup holds at once
constexpr uint32_t LP_TOP = 64;                      // most tokens a row is asked for
constexpr uint32_t LP_POOL = 512;                    // candidates of a block
constexpr uint32_t LP_PARTS = 64;                    // most workgroups a row

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
__device__ __forceinline__ void lp_rebase(LpState& s, float M, float inv_t) {
    if (s.m == M) return;
    const float d = fmaxf((s.m - M) * inv_t, -1e4f), x = __expf(d), l = s.c + s.l;
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
    LpState* states;  // [row][parts]
    uint64_t* keys;   // [row][parts][top]
    uint32_t vocab, top, parts, blocks;  // blocks of LP_BLOCK scores a part
    float inv_t;
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
        if (p.entropy) p.entropy[row] = log_l - s.a / (s.c + s.l);
    }
    if (tid < p.top) {
        const uint64_t k = best[tid];
        p.ids[(size_t)row * p.top + tid] = lp_index(k);
        p.tops[(size_t)row * p.top + tid] = (lp_score(k) - s.m) * p.inv_t - log_l;
    }
}

// The `top` best of pool[0 .. n) to out, best first; 0 where there are fewer. Every thread calls
// it with pool written and waited for; out is to be waited for.
__device__ __forceinline__ void lp_rank(const uint64_t* pool, uint32_t n, uint64_t* out, uint32_t top) {
    for (uint32_t i = threadIdx.x; i < n; i += LP_THREADS) {
        const uint64_t k = pool[i];
        uint32_t rank = 0, j = 0;
        for (; j + 8 <= n; j += 8)  // (the reads of eight do not wait for each other)
#pragma unroll
            for (int e = 0; e < 8; e++) rank += pool[j + e] > k;
        for (; j < n; j++) rank += pool[j] > k;
        if (k != 0 && rank < top) out[rank] = k;
    }
}

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) x = fmaxf(x, __shfl_xor(x, d));
    return x;
}
__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) x += __shfl_xor(x, d);
    return x;
}

struct __attribute__((packed, aligned(4))) Float4Any {  // rows of an odd vocabulary start anywhere
    float x, y, z, w;
};

__global__ __launch_bounds__(LP_THREADS) void k_logprobs(const LpParams p) {
    __shared__ uint64_t pool[LP_TOP + LP_POOL], best[LP_TOP], pick[4];
    __shared__ float red[4][4];
    __shared__ __attribute__((aligned(16))) float gmax[LP_THREADS];
    __shared__ uint32_t count;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row = blockIdx.y, part = blockIdx.x;
    const float* s = p.scores + (size_t)row * p.vocab;
    LpState st{-INFINITY, 0.0f, 0.0f, 0.0f};
    uint32_t kept = 0;  // keys in best
    for (uint32_t b = 0; b < p.blocks; b++) {
        const uint64_t base = ((uint64_t)part * p.blocks + b) * LP_BLOCK;
        if (base >= p.vocab) break;
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
        lp_rebase(st, fmaxf(st.m, top), p.inv_t);
        const float m = st.m == -INFINITY ? 0.0f : st.m;
#pragma unroll
        for (int e = 0; e < LP_EACH; e++) {
            const float x = (v[e] - m) * p.inv_t, w = __expf(x);
            st.l += x == 0.0f ? 0.0f : w;
            st.c += x == 0.0f ? 1.0f : 0.0f;
            st.a += w * fmaxf(x, -1e4f);  // (0 for a score of -inf; a NaN stays one)
        }
        if (p.top == 0) continue;
        // At least `top` of the block's scores reach the top'th largest of its groups' maxima.
        const uint32_t groups = p.top <= 32 ? 64 : LP_THREADS;
        float gm = top;
        if (groups == 64) {  // four threads a group
            gm = fmaxf(gm, __shfl_xor(gm, 1));
            gm = fmaxf(gm, __shfl_xor(gm, 2));
        }
        __syncthreads();  // (the block before has done with gmax, pool and count)
        if (groups == LP_THREADS) gmax[tid] = gm;
        else if ((tid & 3) == 0) gmax[tid >> 2] = gm;
        if (tid == 0) count = kept;
        if (tid < kept) pool[tid] = best[tid];
        __syncthreads();
        // The smallest of those that fewer than `top` are larger than; a wave looks at 64 of them.
        const float mine = gmax[(groups == 64 ? 0 : 64 * wave) + lane];
        uint32_t above = 0;
        for (uint32_t j = 0; j < groups; j += 16)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const float4 x = *(const float4*)&gmax[j + e];
                above += (uint32_t)(x.x > mine) + (uint32_t)(x.y > mine) + (uint32_t)(x.z > mine) + (uint32_t)(x.w > mine);
            }
        float least = -wave_max(above < p.top ? -mine : -INFINITY);
        if (groups != 64) {
            if (lane == 0) red[0][wave] = least;
            __syncthreads();
            least = fminf(fminf(red[0][0], red[0][1]), fminf(red[0][2], red[0][3]));
        }
        // Numbers above -inf (under a mask those alone, if they are enough), and above the worst key
        // kept, whose score beats its equals of later blocks.
        const float worst = kept == p.top ? lp_score(best[p.top - 1]) : -INFINITY, floor = worst != worst ? -INFINITY : worst;
        uint32_t pass = 0;
#pragma unroll
        for (int e = 0; e < LP_EACH; e++) pass |= (uint32_t)(v[e] >= least && v[e] > floor) << e;
        if (__any(pass)) {
            uint32_t at = pass ? atomicAdd(&count, (uint32_t)__popc(pass)) : 0;
#pragma unroll
            for (int e = 0; e < LP_EACH; e++)
                if (pass >> e & 1u) {
                    if (at < LP_TOP + LP_POOL) pool[at] = lp_key(v[e], index(e));
                    at++;
                }
        }
        __syncthreads();
        uint32_t n = count;
        // Candidates that are fewer than asked for may leave out scores of -inf and NaNs.
        const uint32_t here = (uint32_t)min((uint64_t)LP_BLOCK, p.vocab - base);
        const bool few = n < p.top && n - kept < here;
        if (few || n > LP_TOP + LP_POOL) {
            uint32_t taken = 0;
            n = kept;
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
                w = max(max(pick[0], pick[1]), max(pick[2], pick[3]));
                __syncthreads();
                if (w == k && k != 0) {  // (keys are unique: one thread's)
                    const uint32_t off = lp_index(k) - (uint32_t)base;
                    taken |= 1u << (off / (4 * LP_THREADS) * 4 + (off & 3));
                    pool[n] = k;
                }
                n++;
            }
            __syncthreads();
        }
        if (n > kept) {
            lp_rank(pool, n, best, p.top);
            kept = min(n, p.top);
        }
        __syncthreads();
    }
    // The threads' states.
    float M = wave_max(st.m);
    __syncthreads();
    if (lane == 0) red[0][wave] = M;
    __syncthreads();
    M = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    lp_rebase(st, M, p.inv_t);
    st.c = wave_sum(st.c);
    st.l = wave_sum(st.l);
    st.a = wave_sum(st.a);
    if (lane == 0) {
        red[1][wave] = st.c;
        red[2][wave] = st.l;
        red[3][wave] = st.a;
    }
    __syncthreads();
    st = LpState{M, (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]), (red[2][0] + red[2][1]) + (red[2][2] + red[2][3]),
                 (red[3][0] + red[3][1]) + (red[3][2] + red[3][3])};
    if (p.parts == 1) {
        lp_finish(p, row, st, best);
        return;
    }
    const size_t at = (size_t)row * p.parts + part;
    if (tid == 0) p.states[at] = st;
    if (tid < p.top) p.keys[at * p.top + tid] = tid < kept ? best[tid] : 0;
}

__global__ __launch_bounds__(LP_THREADS) void k_logprobs_join(const LpParams p) {
    __shared__ uint64_t pool[LP_PARTS * LP_TOP], best[LP_TOP];
    __shared__ uint64_t low[LP_PARTS];
    __shared__ LpState all;
    __shared__ uint32_t count;
    const uint32_t tid = threadIdx.x, row = blockIdx.x;
    const LpState* states = p.states + (size_t)row * p.parts;
    if (tid < 64) {  // LP_PARTS is a wave
        LpState s = tid < p.parts ? states[tid] : LpState{-INFINITY, 0.0f, 0.0f, 0.0f};
        lp_rebase(s, wave_max(s.m), p.inv_t);
        s.c = wave_sum(s.c);
        s.l = wave_sum(s.l);
        s.a = wave_sum(s.a);
        if (tid == 0) {
            all = s;
            count = 0;
        }
    }
    if (p.top) {
        // Every part's keys are in order: with ceil(top / parts) of each at or above the smallest
        // of those, `top` are.
        const uint64_t* keys = p.keys + (size_t)row * p.parts * p.top;
        const uint32_t each = (p.top + p.parts - 1) / p.parts;
        if (tid < p.parts) low[tid] = keys[tid * p.top + each - 1];
        __syncthreads();
        uint64_t least = low[0];
        for (uint32_t i = 1; i < p.parts; i++) least = min(least, low[i]);
        for (uint32_t i = tid; i < p.parts * p.top; i += LP_THREADS) {
            const uint64_t k = keys[i];
            if (k >= least && k != 0) pool[atomicAdd(&count, 1u)] = k;
        }
        __syncthreads();
        lp_rank(pool, count, best, p.top);
    }
    __syncthreads();
    lp_finish(p, row, all, best);
}

uint32_t lp_parts(uint32_t vocab) { return std::min<uint32_t>(LP_PARTS, (vocab + LP_BLOCK - 1) / LP_BLOCK); }
size_t lp_row_bytes(uint32_t parts, uint32_t top) { return (size_t)parts * (sizeof(LpState) + top * sizeof(uint64_t)); }

}  // namespace

size_t logprobs_scratch_bytes(uint32_t rows, uint32_t vocab, uint32_t top) {
    const uint32_t parts = lp_parts(vocab);
    return parts == 1 ? 0 : rows * lp_row_bytes(parts, top);
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
    p.parts = scratch ? lp_parts(vocab) : 1;
    const uint32_t all = (vocab - 1) / LP_BLOCK + 1;
    p.blocks = (all + p.parts - 1) / p.parts;
    p.inv_t = 1.0f / temperature;
    p.keys = (uint64_t*)scratch;
    p.states = (LpState*)((uint64_t*)scratch + (size_t)rows * p.parts * top);
    hipLaunchKernelGGL(k_logprobs, dim3(p.parts, rows), dim3(LP_THREADS), 0, s, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.parts == 1) return e;
    hipLaunchKernelGGL(k_logprobs_join, dim3(rows), dim3(LP_THREADS), 0, s, p);
    return hipGetLastError();
}

}  // namespace bchip
