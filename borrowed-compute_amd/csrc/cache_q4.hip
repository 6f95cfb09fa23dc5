// What a cache in 4 bits (q4.hpp) needs beside attention: the rotation and append of new rows,
// conversion to and from f32 and f16, and the moves of a cache's rows.
//
// k_rope_append_q4 is k_rope_append (rope.hip) over such a cache: q rotates in place with the
// same expressions, and k, rotated the same, and v go into the cache as codes. A thread takes
// one pair of q heads or two consecutive elements of k or v heads, so sixteen lanes hold a
// block and agree on its scale by four shuffles. Bound by q's traffic for many rows (4096 rows
// of 32 + 2 x 8 heads of 128: 42 us, 4.1 TB/s, of 56 with a sine and cosine for every head; 512
// rows 8.6 us) and by the launch for few (5 us up to 128 rows).
//
// Conversions and moves, bound by memory (1024 elements a slot; the launch, 4 us, up to 512 slots). 131072
// slots: f32 to codes 156 us, 3.9 TB/s read and written; f16 to codes 145, 2.4 TB/s (two elements a lane and a
// byte a store bound both); codes to f32 110 and to f16 62, 5.6 TB/s; codes to codes 26, 5.9 TB/s. Growth of 64
// buffers from 8192 to 16384 slots 156 us, 5.8 TB/s. keep of 8 rows of 64 buffers 12 us and moves, a launch
// for each piece that does not overlap, as over f16 (4096 slots moved down by 4096: 4 us; by 64: 171 us).
#include "common.hpp"
#include "internal.hpp"
#include "q4.hpp"

#include <type_traits>

namespace bchip {

// Pairs of a call from which a thread takes four heads' for one sine and cosine (32 + 2 x 8 heads of 128,
// 1024 rows: 12.1 us against 16.1; 256 rows: 6.7 against 6.0, 28 + 2 x 4 heads, 512 rows: 8.6 against 8.1,
// where the launch has too few threads).
constexpr uint64_t Q4_SHARED_PAIRS = 5 << 18;

struct Q4RowSlots {
    uint64_t slot[MAX_ITEMS];
};

// Row r goes to slot slot0 + r, or (RAGGED) to sl.slot[r]. hd a multiple of 32. A thread takes its
// pair of up to HG heads, whose rotation is the same.
template <bool RAGGED, int HG>
__global__ __launch_bounds__(256) void k_rope_append_q4(float* __restrict__ q, const float* __restrict__ k,
                                                        const float* __restrict__ v, uint8_t* __restrict__ kc,
                                                        uint8_t* __restrict__ vc, const float* __restrict__ inv_freq,
                                                        const uint32_t* __restrict__ positions, uint32_t rows,
                                                        uint32_t nh, uint32_t nkv, uint32_t hd, uint32_t rope_dim,
                                                        uint32_t neox, uint64_t slot0, const Q4RowSlots sl) {
    const uint32_t half = hd / 2, qg = (nh + HG - 1) / HG, kg = (nkv + HG - 1) / HG, groups = qg + 2 * kg;
    const uint64_t idx = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (idx >= (uint64_t)rows * groups * half) return;  // (whole blocks of sixteen lanes: half % 16 == 0)
    const uint32_t p = idx % half, gx = (idx / half) % groups;
    const uint64_t r = idx / ((uint64_t)half * groups);
    if (gx < qg) {
        uint32_t a, b;
        if (!rope_pair(p, rope_dim, neox, a, b)) return;
        float* hp = q + (r * nh + gx * HG) * hd;
        float x[HG][2], s, c;
#pragma unroll
        for (int h = 0; h < HG; h++)
            if (gx * HG + h < nh) x[h][0] = hp[h * hd + a], x[h][1] = hp[h * hd + b];
        sincosf((float)positions[r] * inv_freq[p], &s, &c);
#pragma unroll
        for (int h = 0; h < HG; h++)
            if (gx * HG + h < nh) {
                float y0, y1;
                rotate_sc(x[h][0], x[h][1], s, c, y0, y1);
                hp[h * hd + a] = y0;
                hp[h * hd + b] = y1;
            }
        return;
    }
    const bool isk = gx < qg + kg;
    const uint32_t h0 = (isk ? gx - qg : gx - qg - kg) * HG;
    const float* hp = (isk ? k : v) + (r * nkv + h0) * hd;
    uint8_t* dst = isk ? kc : vc;
    const uint64_t e0 = (RAGGED ? sl.slot[r] : slot0 + r) * ((uint64_t)nkv * hd) + 2 * p;
    // Elements 2p and 2p + 1 of each head: a pair, or (neox) the same half of two pairs.
    const uint32_t hh = rope_dim / 2;
    const float pos = (float)positions[r];
    uint32_t other[2] = {2 * p + 1, 2 * p};
    float s[2] = {0, 0}, c[2] = {1, 1};
    bool first[2] = {true, false}, turn[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const uint32_t e = 2 * p + i;
        turn[i] = isk && e < rope_dim;
        if (neox && turn[i]) {
            first[i] = e < hh;
            other[i] = first[i] ? e + hh : e - hh;
            sincosf(pos * inv_freq[first[i] ? e : e - hh], &s[i], &c[i]);
        }
    }
    if (!neox && turn[0]) {
        sincosf(pos * inv_freq[p], &s[0], &c[0]);
        s[1] = s[0], c[1] = c[0];
    }
    float x[HG][2], y[HG][2];
#pragma unroll
    for (int h = 0; h < HG; h++)
        if (h0 + h < nkv) {
            x[h][0] = hp[h * hd + 2 * p], x[h][1] = hp[h * hd + 2 * p + 1];
            if (neox) {
#pragma unroll
                for (int i = 0; i < 2; i++) y[h][i] = turn[i] ? hp[h * hd + other[i]] : 0.0f;
            } else {
                y[h][0] = x[h][1], y[h][1] = x[h][0];
            }
        }
#pragma unroll
    for (int h = 0; h < HG; h++)
        if (h0 + h < nkv) {
            float z[2];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                float y0, y1;
                rotate_sc(first[i] ? x[h][i] : y[h][i], first[i] ? y[h][i] : x[h][i], s[i], c[i], y0, y1);
                z[i] = !turn[i] ? x[h][i] : first[i] ? y0 : y1;
            }
            uint8_t codes;
            const f16 d = q4_quantise(z[0], z[1], codes);
            const uint64_t e = e0 + (uint64_t)(h0 + h) * hd;
            dst[q4_code_at(e)] = codes;
            if (p % 16 == 0) *(f16*)(dst + q4_scale_at(e)) = d;
        }
}

// dst[off + i] = src[i]: two elements a thread, n and off multiples of 32.
template <typename S>
__global__ __launch_bounds__(256) void k_to_q4(const S* __restrict__ src, uint8_t* __restrict__ dst, uint64_t off,
                                               uint64_t n) {
    // (n / 2 is a multiple of 16 and so is every stride: blocks stay within sixteen lanes.)
    for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n / 2; i += (uint64_t)gridDim.x * blockDim.x) {
        uint8_t codes;
        const f16 d = q4_quantise((float)src[2 * i], (float)src[2 * i + 1], codes);
        const uint64_t e = off + 2 * i;
        dst[q4_code_at(e)] = codes;
        if (i % 16 == 0) *(f16*)(dst + q4_scale_at(e)) = d;
    }
}

// dst[i] = src[i]: eight elements a thread. An f16 holds every value exactly.
template <typename D>
__global__ __launch_bounds__(256) void k_from_q4(const uint8_t* __restrict__ src, D* __restrict__ dst, uint64_t n) {
    for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n / 8; i += (uint64_t)gridDim.x * blockDim.x) {
        const uint32_t w = *(const uint32_t*)(src + q4_code_at(8 * i));
        const float d = (float)*(const f16*)(src + q4_scale_at(8 * i));
#pragma unroll
        for (int j = 0; j < 8; j++) dst[8 * i + j] = (D)(((float)((w >> (4 * j)) & 15u) - 8.0f) * d);
    }
}

// A block's codes and scale.
struct Q4Block {
    uint4 codes;
    uint16_t scale;
};
__device__ __forceinline__ Q4Block q4_block(const uint8_t* b, uint64_t i) {
    return {*(const uint4*)(b + q4_code_at(i * Q4_BLOCK)), *(const uint16_t*)(b + q4_scale_at(i * Q4_BLOCK))};
}
__device__ __forceinline__ void q4_put(uint8_t* b, uint64_t i, const Q4Block& x) {
    *(uint4*)(b + q4_code_at(i * Q4_BLOCK)) = x.codes;
    *(uint16_t*)(b + q4_scale_at(i * Q4_BLOCK)) = x.scale;
}

// dst block to + i = src block from + i, a block a thread; src may be dst where the ranges do
// not overlap.
__global__ __launch_bounds__(256) void k_blocks_q4(const uint8_t* src, uint8_t* dst, uint64_t from, uint64_t to,
                                                   uint64_t n) {
    for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (uint64_t)gridDim.x * blockDim.x)
        q4_put(dst, to + i, q4_block(src, from + i));
}

struct Q4KeepArgs {
    uint8_t* bufs[64];
    uint32_t rows[64];
};

// k_keep (kvcache.hip) with a block a thread: the moves of one block column, in order.
__global__ __launch_bounds__(256) void k_keep_q4(const Q4KeepArgs a, uint32_t nbufs, uint32_t width, uint64_t base,
                                                 uint32_t nrows) {
    const uint32_t col = blockIdx.x * blockDim.x + threadIdx.x;
    if (col >= width || blockIdx.y >= nbufs) return;
    uint8_t* b = a.bufs[blockIdx.y];
    for (uint32_t i = 0; i < nrows; i++) {
        const uint32_t r = a.rows[i];
        if (r != i) q4_put(b, (base + i) * width + col, q4_block(b, (base + r) * width + col));
    }
}

struct Q4GrowArgs {
    const uint8_t* src[64];
    uint8_t* dst[64];
};

// k_grow with a block a thread: the first `keep` blocks copied, zeros behind them.
__global__ __launch_bounds__(256) void k_grow_q4(const Q4GrowArgs a, uint64_t keep, uint64_t total) {
    const uint8_t* src = a.src[blockIdx.y];
    uint8_t* dst = a.dst[blockIdx.y];
    for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (uint64_t)gridDim.x * blockDim.x)
        q4_put(dst, i, i < keep ? q4_block(src, i) : Q4Block{{0u, 0u, 0u, 0u}, 0});
}

static uint32_t blocks_of(uint64_t n) { return (uint32_t)((n + 255) / 256); }
static uint32_t grid_of(uint64_t n) {
    const uint64_t b = (n + 255) / 256;
    return (uint32_t)(b > 65536 ? 65536 : (b ? b : 1));
}

template <int HG>
static hipError_t rope_append_q4_heads(float* q, const float* k, const float* v, void* kc, void* vc, const float* inv_freq,
                                       const uint32_t* positions, uint32_t rows, uint32_t nh, uint32_t nkv, uint32_t hd,
                                       uint32_t rope_dim, uint32_t neox, uint64_t slot0, const uint64_t* slots,
                                       hipStream_t s) {
    const uint64_t per_row = ((nh + HG - 1) / HG + 2 * (uint64_t)((nkv + HG - 1) / HG)) * (hd / 2);
    if (!slots) {
        hipLaunchKernelGGL((k_rope_append_q4<false, HG>), dim3(blocks_of(rows * per_row)), dim3(256), 0, s, q, k, v,
                           (uint8_t*)kc, (uint8_t*)vc, inv_freq, positions, rows, nh, nkv, hd, rope_dim, neox, slot0,
                           Q4RowSlots{});
        return hipGetLastError();
    }
    for (uint32_t r0 = 0; r0 < rows; r0 += MAX_ITEMS) {
        const uint32_t nr = rows - r0 < MAX_ITEMS ? rows - r0 : MAX_ITEMS;
        Q4RowSlots sl{};
        for (uint32_t i = 0; i < nr; i++) sl.slot[i] = slots[r0 + i];
        hipLaunchKernelGGL((k_rope_append_q4<true, HG>), dim3(blocks_of(nr * per_row)), dim3(256), 0, s,
                           q + (size_t)r0 * nh * hd, k + (size_t)r0 * nkv * hd, v + (size_t)r0 * nkv * hd,
                           (uint8_t*)kc, (uint8_t*)vc, inv_freq, positions + r0, nr, nh, nkv, hd, rope_dim, neox, 0ull,
                           sl);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

hipError_t rope_append_q4_launch(float* q, const float* k, const float* v, void* kc, void* vc, const float* inv_freq,
                                 const uint32_t* positions, uint32_t rows, uint32_t nh, uint32_t nkv, uint32_t hd,
                                 uint32_t rope_dim, uint32_t neox, uint64_t slot0, const uint64_t* slots,
                                 hipStream_t s) {
    if (rows == 0) return hipSuccess;
    const uint64_t pairs = (uint64_t)rows * (nh + 2 * (uint64_t)nkv) * (hd / 2);
    const auto launch = pairs >= Q4_SHARED_PAIRS ? rope_append_q4_heads<4> : rope_append_q4_heads<1>;
    return launch(q, k, v, kc, vc, inv_freq, positions, rows, nh, nkv, hd, rope_dim, neox, slot0, slots, s);
}

hipError_t copy_q4_launch(const void* src, uint32_t st, void* dst, uint32_t dt, uint64_t off, uint64_t n,
                          hipStream_t s) {
    if (n == 0) return hipSuccess;
    if (st == 2 && dt == 2)
        hipLaunchKernelGGL(k_blocks_q4, dim3(grid_of(n / Q4_BLOCK)), dim3(256), 0, s, (const uint8_t*)src,
                           (uint8_t*)dst, 0ull, off / Q4_BLOCK, n / Q4_BLOCK);
    else if (dt == 2 && st == 1)
        hipLaunchKernelGGL(k_to_q4<f16>, dim3(grid_of(n / 2)), dim3(256), 0, s, (const f16*)src, (uint8_t*)dst, off, n);
    else if (dt == 2)
        hipLaunchKernelGGL(k_to_q4<float>, dim3(grid_of(n / 2)), dim3(256), 0, s, (const float*)src, (uint8_t*)dst, off,
                           n);
    else if (dt == 1)
        hipLaunchKernelGGL(k_from_q4<f16>, dim3(grid_of(n / 8)), dim3(256), 0, s, (const uint8_t*)src, (f16*)dst + off,
                           n);
    else
        hipLaunchKernelGGL(k_from_q4<float>, dim3(grid_of(n / 8)), dim3(256), 0, s, (const uint8_t*)src,
                           (float*)dst + off, n);
    return hipGetLastError();
}

hipError_t move_q4_launch(void* buf, uint64_t from, uint64_t to, uint64_t n, hipStream_t s) {
    if (n == 0 || from == to) return hipSuccess;
    // Overlapping ranges move in pieces of from - to, as in move_launch.
    const uint64_t f = from / Q4_BLOCK, t = to / Q4_BLOCK, nb = n / Q4_BLOCK, step = f - t < nb ? f - t : nb;
    for (uint64_t o = 0; o < nb; o += step) {
        const uint64_t m = nb - o < step ? nb - o : step;
        hipLaunchKernelGGL(k_blocks_q4, dim3(grid_of(m)), dim3(256), 0, s, (const uint8_t*)buf, (uint8_t*)buf, f + o,
                           t + o, m);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

hipError_t keep_q4_launch(void* const* bufs, uint32_t nbufs, uint32_t width, uint64_t base, const uint32_t* rows,
                          uint32_t nrows, hipStream_t s) {
    if (nbufs == 0 || nrows == 0 || width == 0) return hipSuccess;
    const uint32_t wb = width / Q4_BLOCK;
    for (uint32_t b0 = 0; b0 < nbufs; b0 += 64) {
        Q4KeepArgs a{};
        const uint32_t nb = nbufs - b0 < 64 ? nbufs - b0 : 64;
        for (uint32_t i = 0; i < nb; i++) a.bufs[i] = (uint8_t*)bufs[b0 + i];
        for (uint32_t i = 0; i < nrows; i++) a.rows[i] = rows[i];
        hipLaunchKernelGGL(k_keep_q4, dim3((wb + 255) / 256, nb), dim3(256), 0, s, a, nb, wb, base, nrows);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

hipError_t grow_q4_launch(const void* const* src, void* const* dst, uint32_t nbufs, uint64_t keep, uint64_t total,
                          hipStream_t s) {
    if (nbufs == 0 || total == 0) return hipSuccess;
    for (uint32_t b0 = 0; b0 < nbufs; b0 += 64) {
        Q4GrowArgs a{};
        const uint32_t nb = nbufs - b0 < 64 ? nbufs - b0 : 64;
        for (uint32_t i = 0; i < nb; i++) {
            a.src[i] = (const uint8_t*)src[b0 + i];
            a.dst[i] = (uint8_t*)dst[b0 + i];
        }
        const uint64_t blocks = total / Q4_BLOCK;
        const uint32_t gx = (uint32_t)((blocks + 255) / 256 > 2048 ? 2048 : (blocks + 255) / 256);
        hipLaunchKernelGGL(k_grow_q4, dim3(gx, nb), dim3(256), 0, s, a, keep / Q4_BLOCK, blocks);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace bchip
