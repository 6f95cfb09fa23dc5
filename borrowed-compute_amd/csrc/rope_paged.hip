// RoPE fused with the append to a KV cache in pages, and the copy of whole pages.
//
// k_rope_append_paged: row r's pairs turn by theta = (f32)positions[r] * inv_freq[i], with the
// expressions of k_rope_append (rotate_sc over the device library's full-range sine and cosine), so its
// bits are that kernel's; k and v go to the slot of the row's sequence that the page table names.
// Bound: the bytes of q (read and written), k, v and the slots. A workgroup takes one row, or a part
// of one: its sines and cosines are computed once for all its heads, while the first eight dims of each
// thread are on their way. A thread takes eight dims of a head at a time, 32 bytes, four pairs: neox pairs
// as four dims of either half. 1474 rows of 32 + 2 x 8 heads of 128 into f16 take 14 us, 66 MB at 4.7 TB/s; one
// row 3.5 us, a launch's own latency.
#include "internal.hpp"
#include "paged.hpp"

#include <math.h>

#include <algorithm>

namespace bchip {

namespace {

constexpr uint32_t RP_SEQS = 256;
constexpr uint32_t RP_THREADS = 256;

struct RopePaged {
    float* q;
    const float* k;
    const float* v;
    void* kc;
    void* vc;
    const float* inv_freq;
    const uint32_t* positions;
    const uint32_t* table;
    uint32_t stride, shift, npages, nseq;
    uint32_t nh, nkv, hd, rope_dim, neox;
    uint32_t starts[RP_SEQS + 1], lens[RP_SEQS];
};

template <typename KVT>
__device__ __forceinline__ void put4(KVT* to, f32x4 x);
template <>
__device__ __forceinline__ void put4<float>(float* to, f32x4 x) { *(f32x4*)to = x; }
template <>
__device__ __forceinline__ void put4<f16>(f16* to, f32x4 x) { *(half4*)to = half4{(f16)x[0], (f16)x[1], (f16)x[2], (f16)x[3]}; }

// WIDE: pairs come in fours (rope_dim a multiple of 8); else a thread takes a pair.
template <typename KVT, bool WIDE>
__global__ __launch_bounds__(RP_THREADS) void k_rope_append_paged(const RopePaged p) {
    __shared__ float2 turn[MAX_HD / 2];
    const uint32_t tid = threadIdx.x, lane = tid & 63, row = blockIdx.x;
    // The row's sequence: the last that starts at or before it.
    uint32_t n = 0;
#pragma unroll
    for (uint32_t i = 0; i < RP_SEQS; i += 64) {
        if (i >= p.nseq) break;
        n += __popcll(__ballot(lane + i < p.nseq && p.starts[min(lane + i, RP_SEQS - 1)] <= row));
    }
    const uint32_t seq = __builtin_amdgcn_readfirstlane(n - 1);
    const uint32_t slot = p.lens[seq] - (p.starts[seq + 1] - row);  // (its last rows are the new ones)
    const uint32_t page = p.table[(size_t)seq * p.stride + (slot >> p.shift)];
    const size_t place = (((size_t)page << p.shift) + (slot & ((1u << p.shift) - 1))) * p.nkv * p.hd;
    const uint32_t half = p.rope_dim / 2, per = WIDE ? p.hd / 8 : p.hd / 2, all = (p.nh + 2 * p.nkv) * per;
    const float position = (float)p.positions[row];

    // Where a thread's piece lies: two fours of dims a and b of a head (WIDE), or two dims.
    struct Piece {
        const float* from;
        uint32_t a, b, pair, head;
        bool rot;
    };
    auto piece = [&](uint32_t x) {
        Piece c;
        c.head = x / per;
        const uint32_t i = x - c.head * per;
        const bool isv = c.head >= p.nh + p.nkv;
        c.from = c.head < p.nh ? p.q + ((size_t)row * p.nh + c.head) * p.hd
                               : (isv ? p.v : p.k) + ((size_t)row * p.nkv + c.head - p.nh - (isv ? p.nkv : 0)) * p.hd;
        constexpr uint32_t W = WIDE ? 4 : 1;
        c.rot = !isv && W * i < half;
        c.pair = W * i;
        c.a = c.rot && p.neox ? W * i : 2 * W * i;
        c.b = c.rot && p.neox ? W * i + half : 2 * W * i + W;
        return c;
    };
    typedef typename std::conditional<WIDE, f32x4, float>::type V;
    const uint32_t step = gridDim.y * RP_THREADS;
    uint32_t x = blockIdx.y * RP_THREADS + tid;
    Piece c{};
    V u{}, w{};
    auto get = [&] {
        c = piece(x);
        u = *(const V*)(c.from + c.a);
        w = *(const V*)(c.from + c.b);
    };
    if (x < all) get();
    for (uint32_t i = tid; i < half; i += RP_THREADS) {
        float s, co;
        sincosf(position * p.inv_freq[i], &s, &co);
        turn[i] = float2{s, co};
    }
    __syncthreads();
    while (x < all) {
        if (c.rot) {
            if constexpr (WIDE) {
                float y[8] = {u[0], u[1], u[2], u[3], w[0], w[1], w[2], w[3]};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float2 t = turn[c.pair + e];
                    float z0, z1;
                    rotate_sc(p.neox ? y[e] : e < 2 ? u[2 * e] : w[2 * e - 4], p.neox ? y[e + 4] : e < 2 ? u[2 * e + 1] : w[2 * e - 3], t.x, t.y, z0, z1);
                    if (p.neox) y[e] = z0, y[e + 4] = z1;
                    else y[2 * e] = z0, y[2 * e + 1] = z1;
                }
                u = f32x4{y[0], y[1], y[2], y[3]};
                w = f32x4{y[4], y[5], y[6], y[7]};
            } else {
                const float2 t = turn[c.pair];
                float z0, z1;
                rotate_sc(u, w, t.x, t.y, z0, z1);
                u = z0, w = z1;
            }
        }
        if (c.head < p.nh) {
            if (c.rot) {
                *(V*)(p.q + ((size_t)row * p.nh + c.head) * p.hd + c.a) = u;
                *(V*)(p.q + ((size_t)row * p.nh + c.head) * p.hd + c.b) = w;
            }
        } else if (page < p.npages) {
            const bool isv = c.head >= p.nh + p.nkv;
            KVT* to = (KVT*)(isv ? p.vc : p.kc) + place + (size_t)(c.head - p.nh - (isv ? p.nkv : 0)) * p.hd;
            if constexpr (WIDE) {
                put4<KVT>(to + c.a, u);
                put4<KVT>(to + c.b, w);
            } else {
                to[c.a] = to_kv<KVT>(u);
                to[c.b] = to_kv<KVT>(w);
            }
        }
        x += step;
        if (x < all) get();
    }
}

constexpr uint32_t CP_PAIRS = 256, CP_BUFS = 128, CP_THREADS = 256;
constexpr int CP_EACH = 4;

struct CopyPages {
    uint8_t* bufs[CP_BUFS];
    uint32_t src[CP_PAIRS], dst[CP_PAIRS];
    uint64_t bytes;  // of a page, a multiple of 16
};

// A workgroup moves up to 16 KB of one page in one buffer, four loads a thread on their way. 400 pages of 16 KB in
// 16 buffers take 48 us in two launches, 4.4 TB/s; three pages in 64 buffers 3.6 us.
__global__ __launch_bounds__(CP_THREADS) void k_copy_pages(const CopyPages p) {
    uint8_t* buf = p.bufs[blockIdx.z];
    const uint8_t* from = buf + p.src[blockIdx.y] * p.bytes;
    uint8_t* to = buf + p.dst[blockIdx.y] * p.bytes;
    pg_u32x4 x[CP_EACH];
    const uint64_t at = 16 * ((uint64_t)blockIdx.x * CP_THREADS * CP_EACH + threadIdx.x);
#pragma unroll
    for (int i = 0; i < CP_EACH; i++)  // (past the page: its last piece, not stored)
        x[i] = *(const pg_u32x4*)(from + (at + 16 * CP_THREADS * i < p.bytes ? at + 16 * CP_THREADS * i : p.bytes - 16));
#pragma unroll
    for (int i = 0; i < CP_EACH; i++)
        if (at + 16 * CP_THREADS * i < p.bytes) *(pg_u32x4*)(to + at + 16 * CP_THREADS * i) = x[i];
}

}  // namespace

hipError_t rope_append_paged_launch(float* q, const float* k, const float* v, void* kc, void* vc, uint32_t kv_type,
                                    const float* inv_freq, const uint32_t* positions, const PagedBatch& b, uint32_t nh,
                                    uint32_t nkv, uint32_t hd, uint32_t rope_dim, uint32_t neox, hipStream_t s) {
    const uint32_t rows = b.starts[b.nseq];
    if (rows == 0) return hipSuccess;
    RopePaged p{q, k, v, kc, vc, inv_freq, positions, b.table, b.stride, b.shift, b.npages, b.nseq, nh, nkv, hd, rope_dim, neox, {}, {}};
    std::copy(b.starts, b.starts + b.nseq + 1, p.starts);
    std::copy(b.lens, b.lens + b.nseq, p.lens);
    const bool wide = rope_dim % 8 == 0;
    const uint32_t pieces = (nh + 2 * nkv) * (wide ? hd / 8 : hd / 2);
    // Few rows are shared among workgroups down to a piece a thread.
    const uint32_t most = (pieces + RP_THREADS - 1) / RP_THREADS;
    const uint32_t parts = std::min(std::min(most, 65535u), std::max(1u, 1024u / rows));
    const dim3 grid(rows, parts);
    if (kv_type == 1 && wide) hipLaunchKernelGGL((k_rope_append_paged<f16, true>), grid, dim3(RP_THREADS), 0, s, p);
    else if (kv_type == 1) hipLaunchKernelGGL((k_rope_append_paged<f16, false>), grid, dim3(RP_THREADS), 0, s, p);
    else if (wide) hipLaunchKernelGGL((k_rope_append_paged<float, true>), grid, dim3(RP_THREADS), 0, s, p);
    else hipLaunchKernelGGL((k_rope_append_paged<float, false>), grid, dim3(RP_THREADS), 0, s, p);
    return hipGetLastError();
}

hipError_t copy_pages_launch(void* const* bufs, uint32_t nbufs, uint64_t page_bytes, const uint32_t* src, const uint32_t* dst,
                             uint32_t n, hipStream_t s) {
    const uint64_t each = 16ull * CP_THREADS * CP_EACH;
    for (uint32_t b0 = 0; b0 < nbufs; b0 += CP_BUFS)
        for (uint32_t i0 = 0; i0 < n; i0 += CP_PAIRS) {
            CopyPages p{};
            const uint32_t nb = std::min(CP_BUFS, nbufs - b0), np = std::min(CP_PAIRS, n - i0);
            for (uint32_t i = 0; i < nb; i++) p.bufs[i] = (uint8_t*)bufs[b0 + i];
            std::copy(src + i0, src + i0 + np, p.src);
            std::copy(dst + i0, dst + i0 + np, p.dst);
            p.bytes = page_bytes;
            hipLaunchKernelGGL(k_copy_pages, dim3((uint32_t)((page_bytes + each - 1) / each), np, nb), dim3(CP_THREADS), 0, s, p);
            const hipError_t e = hipGetLastError();
            if (e != hipSuccess) return e;
        }
    return hipSuccess;
}

}  // namespace bchip
