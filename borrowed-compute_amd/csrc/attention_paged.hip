// Attention over a cache in pages (paged.hpp) of many query rows a KV head: prompts, pieces of them,
// verify passes; the fold of chunks, and the plan of a call.
//
// Mathematics and layout as in paged_row.hpp. A workgroup takes 64 or 128 query rows of one
// KV head and its waves share each tile of K and V, two of which are in LDS: the next one arrives
// while this one is computed.
#include "internal.hpp"
#include "paged.hpp"
#include "paged_launch.hpp"
#include "paged_row.hpp"
#include "parts.hpp"

#include <math.h>
#include <stdlib.h>

#include <algorithm>
#include <vector>

namespace bchip {

namespace {

// A block of query rows: q0 .. q1 - 1 of a KV head's (rows x G), its tiles t0 .. t1 - 1.
struct PgBlock {
    uint32_t kvh, q0, q1, r0, h0, seen, end, nchunk, t0, t1;
    size_t unit;  // of its first 16 query rows' states
    size_t next;  // from 16 query rows to the next
};

template <uint32_t QT, uint32_t SLOTS>
__device__ __forceinline__ PgBlock block_of(const PgParams& p, const PgItem& it, uint32_t kvh, uint32_t block) {
    PgBlock b;
    const uint32_t rows = it.rows_seq >> 8, nq = rows * p.G, nqt = (nq - 1) / QT + 1, local = block - it.block0;
    b.kvh = kvh;
    const uint32_t qt = nqt - 1 - local % nqt, chunk = local / nqt;  // the longest lists first
    b.q0 = qt * QT;
    b.q1 = min(b.q0 + QT, nq);
    b.r0 = b.q0 / p.G;
    b.h0 = b.q0 - b.r0 * p.G;
    b.seen = it.len - rows + b.r0 + 1;                // slots that every row here sees,
    b.end = it.len - rows + (b.q1 - 1) / p.G + 1;     // and the last one
    b.nchunk = ((it.len - 1) / SLOTS) / p.tchunk + 1;
    const uint32_t all = (b.end - 1) / SLOTS + 1;
    b.t0 = min(chunk * p.tchunk, all);
    b.t1 = min(b.t0 + p.tchunk, all);
    b.next = b.nchunk;
    b.unit = (size_t)p.blocks * p.nkv + ((size_t)it.block0 * p.nkv + (size_t)b.kvh * nqt * b.nchunk + (size_t)qt * b.nchunk) * (QT / 16) + chunk;
    return b;
}

// A block's 16 query rows from `first`: this lane's row.
struct PgRow {
    bool valid;
    uint32_t vis;  // slots it sees
    size_t at;     // its elements of q and out
};
__device__ __forceinline__ PgRow row_of(const PgParams& p, const PgItem& it, const PgBlock& b, uint32_t i) {
    const uint32_t y = b.h0 + i, dr = (y * (65536 / p.G + 1)) >> 16;  // y / G
    const bool valid = b.q0 + i < b.q1;
    const uint32_t row = it.row0 + b.r0 + (valid ? dr : 0), head = b.kvh * p.G + (valid ? y - dr * p.G : 0);
    return PgRow{valid, valid ? b.seen + dr : b.end, ((size_t)row * p.nh + head) * p.hd};
}

// Every wave's LDS writes and reads are done, its loads have arrived.
__device__ __forceinline__ void tile_barrier() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Bytes of LDS of a workgroup: two tiles of K and V each (f32 in parts: half as much again).
template <typename KVT, int NB>
constexpr uint32_t PG_TILE_LDS = (sizeof(KVT) == 2 ? 16 : 8) * PgTile<KVT, NB>::GRANULE + 16;
template <int NB>
constexpr uint32_t PG_TILE3_LDS = 12 * PgTile<float, NB>::GRANULE + 16;

// f16 caches. RT 2: four waves of 32 query rows; RT 1: eight waves, four of them 16 query rows each over
// half of a tile's slots and four the same rows over the other half. Bound by the matrix cores where rows are
// many: 2048 before 8192 slots, 32 x 8 heads of 128, take 509 to 527 us by card, 1174 to 1214 TFLOP/s with both
// parts of q and of the weights (a large library product in f16 reaches 1132); 600 before 2000 63 us, of which the
// last blocks and the fold's 8.8 us are a third.
// Block `id` of the items of more than 16 query rows. lds: PG_TILE_LDS bytes, 16-byte aligned.
template <int NB, int RT>
__device__ __forceinline__ void tile16_block(const PgParams& p, uint32_t id, uint8_t* lds) {
    using T = PgTile<f16, NB>;
    constexpr int NF = 2 * NB, KS = RT == 1 ? 2 : 1;
    constexpr uint32_t QT = 64 * RT, SLOTS = 64;
    uint8_t(*kt)[4 * T::GRANULE] = (uint8_t(*)[4 * T::GRANULE])lds, (*vt)[4 * T::GRANULE] = (uint8_t(*)[4 * T::GRANULE])(lds + 8 * T::GRANULE);
    uint32_t* odd_tile = (uint32_t*)(lds + 16 * T::GRANULE);  // 1 + the tile of each buffer whose V holds an infinity or a NaN
    static_assert(KS == 1 || 8 * T::GRANULE >= sizeof(f32x4) * 4 * NF * 64, "the second waves' states");
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((threadIdx.x >> 6) & 3);
    const uint32_t ks = __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
    const uint32_t m16 = lane & 15, g = lane >> 4;
    const uint32_t block = id / p.nkv;
    uint32_t which;
    const PgItem it = item_with_arguments<false>(p, false, block, which);
    const PgBlock b = block_of<QT, SLOTS>(p, it, id % p.nkv, block);
    if (b.t0 >= b.t1) {  // nothing of these rows' lists
        if (threadIdx.x < QT) {
            const size_t u = b.unit + threadIdx.x / 16 * b.next;
            *(float2*)(p.part_ml + 2 * (u * 16 + (threadIdx.x & 15))) = float2{-INFINITY, 0.0f};
        }
        return;
    }
    PgList list = list_of(p, it, b.kvh, 2);
    list.end = b.end;

    // A wave brings granule `wave` of a tile, K's and V's (KS 2: K's or V's).
    uint32_t kfrom[T::LOADS], vfrom[KS == 1 ? T::LOADS : 1], page;
#pragma unroll
    for (int i = 0; i < T::LOADS; i++) {
        kfrom[i] = KS == 2 && ks ? T::template from<true>(i, lane, list.row_bytes, p.hd * 2) : T::template from<false>(i, lane, list.row_bytes, p.hd * 2);
        if constexpr (KS == 1) vfrom[i] = T::template from<true>(i, lane, list.row_bytes, p.hd * 2);
    }
    const uint32_t kl = (uint32_t)(uintptr_t)(pg_lds*)&kt[0][0], vl = (uint32_t)(uintptr_t)(pg_lds*)&vt[0][0];
    auto look = [&](uint32_t t) { page = list.page(t * SLOTS + 16 * wave); };
    auto fetch = [&](uint32_t t, uint32_t buf) {
        const uint32_t slot = t * SLOTS + 16 * wave, at = buf * 4 * T::GRANULE + wave * T::GRANULE;
        const bool k = KS == 1 || !ks, v = KS == 1 || ks;
        if (k && list.bad(slot, page)) {  // a page past the pool: the rows that see its slots are NaN
#pragma unroll
            for (int i = 0; i < T::LOADS; i++) *(pg_u32x4*)(&kt[0][0] + at + 1024 * i + 16 * lane) = pg_u32x4{0x7e007e00u, 0x7e007e00u, 0x7e007e00u, 0x7e007e00u};
        } else if (k) {
            const pg_u32x4 r = list.granule(p.kc, slot, page);
#pragma unroll
            for (int i = 0; i < T::LOADS; i++) load_lds(r, kfrom[i], kl + at, 1024 * i);
        }
        if (v) {
            const pg_u32x4 r = list.granule(p.vc, slot, page);
#pragma unroll
            for (int i = 0; i < T::LOADS; i++) load_lds(r, KS == 1 ? vfrom[KS == 1 ? i : 0] : kfrom[i], vl + at, 1024 * i);
        }
    };
    look(b.t0);
    if (threadIdx.x < 2) odd_tile[threadIdx.x] = 0;

    PgRow row[RT];
    half8 qh[RT][NB], ql[RT][NB];
    float c[RT];
    {
        f32x4 y[RT][NB][2];
#pragma unroll
        for (int r = 0; r < RT; r++) {
            row[r] = row_of(p, it, b, (wave * RT + r) * 16 + m16);
#pragma unroll
            for (int j = 0; j < NB; j++)  // (no branch around them)
#pragma unroll
                for (int e = 0; e < 2; e++) y[r][j][e] = *(const f32x4*)(p.q + row[r].at + (32 * j + 8 * g < p.hd ? 32 * j + 8 * g : 0) + 4 * e);
        }
        // They are waited for here, beside the page: behind the tile's loads, which the compiler does not
        // count, its wait for them would be one for those too.
#pragma unroll
        for (int r = 0; r < RT; r++)
#pragma unroll
            for (int j = 0; j < NB; j++)
#pragma unroll
                for (int e = 0; e < 2; e++) asm volatile("" : "+v"(y[r][j][e]));
        fetch(b.t0, 0);
        look(b.t0 + 1);
#pragma unroll
        for (int r = 0; r < RT; r++) {
            float top = 0.0f, k, x[NB][8];
#pragma unroll
            for (int j = 0; j < NB; j++) {
#pragma unroll
                for (int e = 0; e < 8; e++) x[j][e] = row[r].valid && 32 * j + 8 * g < p.hd ? y[r][j][e >> 2][e & 3] : 0.0f;
                top = q_top(x[j], top);
            }
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            q_scale(top, p.sc, k, c[r]);
#pragma unroll
            for (int j = 0; j < NB; j++) q_parts(x[j], k, qh[r][j], ql[r][j]);
        }
    }
    uint32_t kat[NB], vat[NF];
#pragma unroll
    for (int j = 0; j < NB; j++) kat[j] = T::at(m16, 4 * j + g, T::turn_k(m16));
    {
        const uint32_t slot = 4 * g + (m16 >> 2);
#pragma unroll
        for (int f = 0; f < NF; f++) vat[f] = T::at(slot, 2 * f + ((m16 >> 1) & 1), T::turn_v(slot)) + 8 * (m16 & 1);
    }

    f32x4 o[RT][NF];
    float ref[RT], l[RT];
#pragma unroll
    for (int r = 0; r < RT; r++) {
        ref[r] = -INFINITY;
        l[r] = 0.0f;
#pragma unroll
        for (int f = 0; f < NF; f++) o[r][f] = f32x4{0, 0, 0, 0};
    }
    for (uint32_t t = b.t0; t < b.t1; t++) {
        const uint32_t buf = (t - b.t0) & 1, ts = t * SLOTS;
        tile_barrier();
        if (t + 1 < b.t1) {
            fetch(t + 1, buf ^ 1);
            look(t + 2);
        }
        const uint8_t *kb = kt[buf], *vb = vt[buf];
        const bool edge = ts + SLOTS > b.seen;
        if (edge && b.seen < b.end) {
            // Some row does not see all of the tile: an infinity or a NaN in V, which a weight of 0
            // would not silence, reaches the rows that see its slot and is 0 from then on.
            // (The threads' last round may reach past the tile: heads of 32 and 96 dims by eight waves.)
            constexpr uint32_t BYTES = 4 * T::GRANULE, ROUND = 16 * 256 * KS;
            constexpr bool WHOLE_ROUNDS = BYTES % ROUND == 0;
            bool odd = false;
#pragma unroll
            for (uint32_t from = 0; from < BYTES; from += ROUND) {
                const uint32_t x = from + 16 * threadIdx.x;
                if (!WHOLE_ROUNDS && x >= BYTES) break;
                const pg_u32x4 w = *(const pg_u32x4*)(vb + x);
                odd = odd || odd16(w.x) || odd16(w.y) || odd16(w.z) || odd16(w.w);
            }
            if (odd) odd_tile[buf] = t + 1;
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
            if (odd_tile[buf] == t + 1) {
                for (uint32_t i = KS == 2 ? 32 * ks : 0; i < (KS == 2 ? 32 * ks + 32 : 64u); i++)
#pragma unroll
                    for (int f = 0; f < NF; f++) {
                        const half4 v = *(const half4*)(vb + (i >> 4) * T::GRANULE + T::at(i & 15, 2 * f + (g >> 1), T::turn_v(i)) + 8 * (g & 1));
#pragma unroll
                        for (int r = 0; r < RT; r++)
                            if (ts + i < row[r].vis)
#pragma unroll
                                for (int e = 0; e < 4; e++)
                                    if (odd16(__builtin_bit_cast(uint16_t, v[e]))) o[r][f][e] = NAN;
                    }
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
                __builtin_amdgcn_s_barrier();
                __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
                for (uint32_t x = 16 * threadIdx.x; x < BYTES; x += ROUND) {
                    pg_u32x4* at = (pg_u32x4*)(vb + x);
                    pg_u32x4 w = *at;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        if ((w[e] & 0x7c00u) == 0x7c00u) w[e] &= 0xffff0000u;
                        if ((w[e] & 0x7c000000u) == 0x7c000000u) w[e] &= 0xffffu;
                    }
                    *at = w;
                }
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
                __builtin_amdgcn_s_barrier();
                __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
            }
        }
#pragma unroll
        for (int i = 0; i < 2 / KS; i++) {
            const uint32_t u = KS == 2 ? ks : i;  // 32 of the tile's slots
            // (Four sums in turn, so that no MFMA waits for the one before: one set of rows takes the
            // parts of q apart.)
            constexpr bool APART = RT == 1;
            f32x4 s[RT][2], s2[2];
#pragma unroll
            for (int r = 0; r < RT; r++) s[r][0] = s[r][1] = s2[0] = s2[1] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < NB; j++) {
                const half8 k0 = *(const half8*)(kb + 2 * u * T::GRANULE + kat[j]), k1 = *(const half8*)(kb + (2 * u + 1) * T::GRANULE + kat[j]);
#pragma unroll
                for (int r = 0; r < RT; r++) {
                    s[r][0] = mfma16(k0, qh[r][j], s[r][0]);
                    s[r][1] = mfma16(k1, qh[r][j], s[r][1]);
                }
#pragma unroll
                for (int r = 0; r < RT; r++) {
                    f32x4(&to)[2] = APART ? s2 : s[r];
                    to[0] = mfma16(k0, ql[r][j], to[0]);
                    to[1] = mfma16(k1, ql[r][j], to[1]);
                }
            }
            half8 ph[RT], pl[RT];
#pragma unroll
            for (int r = 0; r < RT; r++) {
                if (APART) {
                    s[r][0] += s2[0];
                    s[r][1] += s2[1];
                }
                if (edge)
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        if (ts + 32 * u + 16 * (e >> 2) + 4 * g + (e & 3) >= row[r].vis) s[r][e >> 2][e & 3] = -INFINITY;
                float f;
                if (raise(s[r], c[r], ref[r], f)) {
                    l[r] *= f;
#pragma unroll
                    for (int k = 0; k < NF; k++) o[r][k] *= f;
                }
                weights<false>(s[r], c[r], ref[r], 0.0f, l[r], ph[r], pl[r]);
            }
            const uint8_t* vu = vb + 2 * u * T::GRANULE;
#pragma unroll
            for (int f = 0; f < NF; f += 2) {
                half8 v[2];
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const half4 x = read_transposed(vu + vat[f + e]), y = read_transposed(vu + T::GRANULE + vat[f + e]);
                    v[e] = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
                }
#pragma unroll
                for (int r = 0; r < RT; r++) {
                    o[r][f] = mfma16(v[0], ph[r], o[r][f]);
                    o[r][f + 1] = mfma16(v[1], ph[r], o[r][f + 1]);
                }
#pragma unroll
                for (int r = 0; r < RT; r++) {
                    o[r][f] = mfma16(v[0], pl[r], o[r][f]);
                    o[r][f + 1] = mfma16(v[1], pl[r], o[r][f + 1]);
                }
            }
        }
    }

    if constexpr (KS == 2) {  // the two halves of the slots
        f32x4(*so)[NF][64] = (f32x4(*)[NF][64])kt;
        float(*sr)[2][64] = (float(*)[2][64])vt;
        __syncthreads();
        if (ks) {
            sr[wave][0][lane] = ref[0];
            sr[wave][1][lane] = l[0];
#pragma unroll
            for (int f = 0; f < NF; f++) so[wave][f][lane] = o[0][f];
        }
        __syncthreads();
        if (ks) return;
        const float other = sr[wave][0][lane], R2 = fmaxf(ref[0], other), Rs = R2 == -INFINITY ? 0.0f : R2;
        const float a = exp2_hw(ref[0] - Rs), e = exp2_hw(other - Rs);
        ref[0] = R2;
        l[0] = l[0] * a + sr[wave][1][lane] * e;
#pragma unroll
        for (int f = 0; f < NF; f++) o[0][f] = o[0][f] * a + so[wave][f][lane] * e;
    }
#pragma unroll
    for (int r = 0; r < RT; r++) {
        l[r] += __shfl_xor(l[r], 16);
        l[r] += __shfl_xor(l[r], 32);
        if (!row[r].valid) continue;
        if (b.nchunk > 1) {
            const size_t u = b.unit + (wave * RT + r) * b.next;
            f32x4* part = (f32x4*)p.part_o + u * NF * 64 + lane;
#pragma unroll
            for (int f = 0; f < NF; f++) part[64 * f] = o[r][f];
            if (g == 0) *(float2*)(p.part_ml + 2 * (u * 16 + m16)) = float2{ref[r], l[r]};
            continue;
        }
        const float k = 1.0f / l[r];
#pragma unroll
        for (int f = 0; f < NF; f++) {
            const uint32_t d = 16 * f + 4 * g;
            if (d < p.hd) *(f32x4*)(p.out + row[r].at + d) = o[r][f] * k;
        }
    }
}

// f32 caches, on the f32 matrix cores: four waves of 16 query rows, tiles of 32 slots. For few query rows (verify
// passes of 6 rows before 5000 slots: 32 us, by tile3_block's parts in four waves 37), and for heads past 128
// dims, whose parts leave no room for a second wave (8 x 4 heads of 256, 777 rows: 84 us, 88).
template <int NB>
__device__ __forceinline__ void tile32_block(const PgParams& p, uint32_t id, uint8_t* lds) {
    using T = PgTile<float, NB>;
    constexpr int NF = 2 * NB, NJ = 2 * NB, NS = NB / 2, TAIL = NB % 2;
    constexpr uint32_t QT = 64, SLOTS = 32;
    uint8_t(*kt)[2 * T::GRANULE] = (uint8_t(*)[2 * T::GRANULE])lds, (*vt)[2 * T::GRANULE] = (uint8_t(*)[2 * T::GRANULE])(lds + 4 * T::GRANULE);
    uint32_t* odd_tile = (uint32_t*)(lds + 8 * T::GRANULE);
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t m16 = lane & 15, g = lane >> 4;
    const uint32_t block = id / p.nkv;
    uint32_t which;
    const PgItem it = item_with_arguments<false>(p, false, block, which);
    const PgBlock b = block_of<QT, SLOTS>(p, it, id % p.nkv, block);
    if (b.t0 >= b.t1) {
        if (threadIdx.x < QT) {
            const size_t u = b.unit + threadIdx.x / 16 * b.next;
            *(float2*)(p.part_ml + 2 * (u * 16 + (threadIdx.x & 15))) = float2{-INFINITY, 0.0f};
        }
        return;
    }
    PgList list = list_of(p, it, b.kvh, 4);
    list.end = b.end;

    // Two waves bring a tile's two granules of K, two V's.
    const uint32_t half = wave & 1;
    uint32_t from[T::LOADS], page;
#pragma unroll
    for (int i = 0; i < T::LOADS; i++)
        from[i] = wave < 2 ? T::template from<false>(i, lane, list.row_bytes, p.hd * 4) : T::template from<true>(i, lane, list.row_bytes, p.hd * 4);
    const uint32_t kl = (uint32_t)(uintptr_t)(pg_lds*)&kt[0][0], vl = (uint32_t)(uintptr_t)(pg_lds*)&vt[0][0];
    auto look = [&](uint32_t t) { page = list.page(t * SLOTS + 16 * half); };
    auto fetch = [&](uint32_t t, uint32_t buf) {
        const uint32_t slot = t * SLOTS + 16 * half, at = buf * 2 * T::GRANULE + half * T::GRANULE;
        if (wave < 2 && list.bad(slot, page)) {  // a page past the pool: the rows that see its slots are NaN
#pragma unroll
            for (int i = 0; i < T::LOADS; i++) *(f32x4*)(&kt[0][0] + at + 1024 * i + 16 * lane) = f32x4{NAN, NAN, NAN, NAN};
        } else {
            const pg_u32x4 r = list.granule(wave < 2 ? p.kc : p.vc, slot, page);
            const uint32_t to = (wave < 2 ? kl : vl) + at;
#pragma unroll
            for (int i = 0; i < T::LOADS; i++) load_lds(r, from[i], to, 1024 * i);
        }
    };
    look(b.t0);
    if (threadIdx.x < 2) odd_tile[threadIdx.x] = 0;
    const PgRow row = row_of(p, it, b, wave * 16 + m16);
    f32x4 q[NJ];
#pragma unroll
    for (int j = 0; j < NJ; j++) q[j] = *(const f32x4*)(p.q + row.at + (16 * j + 4 * g < p.hd ? 16 * j + 4 * g : 0));
#pragma unroll
    for (int j = 0; j < NJ; j++) asm volatile("" : "+v"(q[j]));  // (as in attn_paged_tile16)
    fetch(b.t0, 0);
    look(b.t0 + 1);
#pragma unroll
    for (int j = 0; j < NJ; j++)
        if (!row.valid || 16 * j + 4 * g >= p.hd) q[j] = f32x4{0, 0, 0, 0};
    uint32_t kat[NJ];
#pragma unroll
    for (int j = 0; j < NJ; j++) kat[j] = T::at(m16, 4 * j + g, T::turn_k(m16));

    f32x4 o[NF];
#pragma unroll
    for (int f = 0; f < NF; f++) o[f] = f32x4{0, 0, 0, 0};
    float ref = -INFINITY, l = 0.0f;
    for (uint32_t t = b.t0; t < b.t1; t++) {
        const uint32_t buf = (t - b.t0) & 1, ts = t * SLOTS;
        tile_barrier();
        if (t + 1 < b.t1) {
            fetch(t + 1, buf ^ 1);
            look(t + 2);
        }
        const uint8_t *kb = kt[buf], *vb = vt[buf];
        const bool edge = ts + SLOTS > b.seen;
        if (edge && b.seen < b.end) {  // (as in attn_paged_tile16)
            constexpr int EACH = 2 * T::GRANULE / (16 * 256);
            static_assert(EACH * 16 * 256 == 2 * T::GRANULE, "a share for every thread");
            bool odd = false;
#pragma unroll
            for (int i = 0; i < EACH; i++) {
                const pg_u32x4 w = *(const pg_u32x4*)(vb + 16 * (threadIdx.x + 256 * i));
                odd = odd || odd32(w.x) || odd32(w.y) || odd32(w.z) || odd32(w.w);
            }
            if (odd) odd_tile[buf] = t + 1;
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
            if (odd_tile[buf] == t + 1) {
                for (uint32_t i = 0; i < SLOTS && ts + i < row.vis; i++)
#pragma unroll
                    for (int f = 0; f < NF; f++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            if (odd32(*(const uint32_t*)(vb + i * T::PITCH + 4 * dim_of<float, NB>(f, g, e)))) o[f][e] = NAN;
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
                __builtin_amdgcn_s_barrier();
                __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
                for (int i = 0; i < EACH; i++) {
                    pg_u32x4* at = (pg_u32x4*)(vb + 16 * (threadIdx.x + 256 * i));
                    pg_u32x4 w = *at;
#pragma unroll
                    for (int e = 0; e < 4; e++) w[e] = odd32(w[e]) ? 0u : w[e];
                    *at = w;
                }
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
                __builtin_amdgcn_s_barrier();
                __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
            }
        }
        f32x4 s[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            f32x4 a[4] = {};
#pragma unroll
            for (int j = 0; j < NJ; j++) {
                const f32x4 k = *(const f32x4*)(kb + h * T::GRANULE + kat[j]);
#pragma unroll
                for (int e = 0; e < 4; e++) a[e] = mfma_f32(k[e], q[j][e], a[e]);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                s[h][i] = ((a[0][i] + a[1][i]) + (a[2][i] + a[3][i])) * p.sc;
                if (edge && ts + 16 * h + 4 * g + i >= row.vis) s[h][i] = -INFINITY;
            }
        }
        float f;
        if (raise(s, 1.0f, ref, f)) {
            l *= f;
#pragma unroll
            for (int k = 0; k < NF; k++) o[k] *= f;
        }
        const float base = ref == -INFINITY ? 0.0f : ref;
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                s[h][i] = exp2_hw(s[h][i] - base);
                l += s[h][i];
            }
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint8_t* at = vb + (16 * h + 4 * g + i) * T::PITCH;
#pragma unroll
                for (int z = 0; z < NS; z++) {
                    const f32x4 v = *(const f32x4*)(at + 256 * z + 16 * m16);
#pragma unroll
                    for (int e = 0; e < 4; e++) o[4 * z + e] = mfma_f32(v[e], s[h][i], o[4 * z + e]);
                }
                if constexpr (TAIL) {
                    const f32x2 v = *(const f32x2*)(at + 256 * NS + 8 * m16);
#pragma unroll
                    for (int e = 0; e < 2; e++) o[4 * NS + e] = mfma_f32(v[e], s[h][i], o[4 * NS + e]);
                }
            }
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (!row.valid) return;
    if (b.nchunk > 1) {
        const size_t u = b.unit + wave * b.next;
        f32x4* part = (f32x4*)p.part_o + u * NF * 64 + lane;
#pragma unroll
        for (int f = 0; f < NF; f++) part[64 * f] = o[f];
        if (g == 0) *(float2*)(p.part_ml + 2 * (u * 16 + m16)) = float2{ref, l};
        return;
    }
    const float k = 1.0f / l;
#pragma unroll
    for (int z = 0; z < NS; z++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t d = 64 * z + 16 * g + 4 * i;
            if (d < p.hd) *(f32x4*)(p.out + row.at + d) = f32x4{o[4 * z][i], o[4 * z + 1][i], o[4 * z + 2][i], o[4 * z + 3][i]} * k;
        }
    if constexpr (TAIL)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t d = 64 * NS + 8 * g + 2 * i;
            if (d < p.hd) *(f32x2*)(p.out + row.at + d) = f32x2{o[4 * NS][i], o[4 * NS + 1][i]} * k;
        }
}

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// Two numbers as three bf16 each, which add up to them: the first cut off after eight bits (so the largest
// stay finite), the second rounded, the third what is left.
__device__ __forceinline__ void split3(float a, float b, uint32_t& h, uint32_t& m, uint32_t& l) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const uint32_t x = __float_as_uint(a), y = __float_as_uint(b);
    h = __builtin_amdgcn_perm(y, x, 0x07060302);
    a -= __uint_as_float(x & 0xffff0000u);
    b -= __uint_as_float(y & 0xffff0000u);
    m = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
    a -= __uint_as_float(m << 16);
    b -= __uint_as_float(m & 0xffff0000u);
    l = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302);
}
__device__ __forceinline__ void split3(const float (&x)[8], bf16x8 (&to)[3]) {
    pg_u32x4 w[3];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint32_t h, m, l;
        split3(x[2 * i], x[2 * i + 1], h, m, l);
        w[0][i] = h, w[1][i] = m, w[2][i] = l;
    }
#pragma unroll
    for (int i = 0; i < 3; i++) to[i] = __builtin_bit_cast(bf16x8, w[i]);
}
__device__ __forceinline__ f32x4 mfma_bf16(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// f32 caches, many query rows: K, V, q and the weights are three bf16 each (24 bits, f32's range), and of their
// nine products the six down to 2^-16 of the first are formed: what is left out is under 2^-22 of a
// product, and the six take 3/8 of the time of one on the f32 matrix cores. Eight waves of 16 query rows, tiles
// of 32 slots, which come through registers: each is cut into its parts, into LDS, while the one before is
// computed, its successor's on their way. Bound by the matrix cores: 2048 rows before 6000 slots, 32 x 8
// heads of 128, take 1.22 ms, 194 TFLOP/s of the formula (1.85 ms on the f32 cores, in tile32_block); 777
// rows before 300 77 us (127). Four waves of 32 query rows read half as much LDS, but alone on their SIMD
// hide less: 88 us where these take 77.
template <int NB>
__device__ __forceinline__ void tile3_block(const PgParams& p, uint32_t id, uint8_t* lds) {
    using P = PgTile<f16, NB>;  // of a part
    constexpr int NF = 2 * NB;
    constexpr uint32_t QT = 128, SLOTS = 32, PIECES = NB;  // a wave's loads, half a granule
    constexpr uint32_t KV = 6 * P::GRANULE, STAGE = 2 * KV;        // [K, V][granule][part]
    uint32_t* odd_tile = (uint32_t*)(lds + 2 * STAGE);        // 1 + the tile of each stage whose V holds an infinity or a NaN
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t m16 = lane & 15, g = lane >> 4;
    const uint32_t block = id / p.nkv;
    uint32_t which;
    const PgItem it = item_with_arguments<false>(p, false, block, which);
    const PgBlock b = block_of<QT, SLOTS>(p, it, id % p.nkv, block);
    if (b.t0 >= b.t1) {
        if (threadIdx.x < QT) {
            const size_t u = b.unit + threadIdx.x / 16 * b.next;
            *(float2*)(p.part_ml + 2 * (u * 16 + (threadIdx.x & 15))) = float2{-INFINITY, 0.0f};
        }
        return;
    }
    PgList list = list_of(p, it, b.kvh, 4);
    list.end = b.end;

    // Four waves bring a tile's two granules of K, half a granule each, four V's.
    const uint32_t half = wave & 1, isv = (wave >> 1) & 1;
    const uint8_t* cache = isv ? p.vc : p.kc;
    uint32_t from[PIECES], to[PIECES], page;
#pragma unroll
    for (uint32_t i = 0; i < PIECES; i++) {
        const uint32_t x = 64 * (i + (wave >> 2) * PIECES) + lane, slot = x / (8 * NB), four = x % (8 * NB);
        from[i] = 4 * four < p.hd ? slot * list.row_bytes + 16 * four : 0x80000000u;
        to[i] = isv * KV + half * 3 * P::GRANULE + P::at(slot, four / 2, isv ? P::turn_v(slot) : P::turn_k(slot)) + 8 * (four & 1);
    }
    auto look = [&](uint32_t t) { page = list.page(t * SLOTS + 16 * half); };
    pg_u32x4 in[PIECES];  // the next tile's,
    bool bad;             // whose page is past the pool
    auto source = [&](uint32_t t) { return list.buffer(cache, t < b.t1 ? t * SLOTS + 16 * half : list.end, page); };
    auto load = [&](__amdgpu_buffer_rsrc_t r, uint32_t i) { in[i] = __builtin_amdgcn_raw_buffer_load_b128(r, from[i], 0, 0); };
    auto put = [&](uint32_t i, uint8_t* stage) {
        u32x2 h, m, l;
#pragma unroll
        for (int e = 0; e < 2; e++) {
            uint32_t x, y, z;
            split3(__uint_as_float(in[i][2 * e]), __uint_as_float(in[i][2 * e + 1]), x, y, z);
            h[e] = x, m[e] = y, l[e] = z;
        }
        *(u32x2*)(stage + to[i]) = h;
        *(u32x2*)(stage + to[i] + P::GRANULE) = m;
        *(u32x2*)(stage + to[i] + 2 * P::GRANULE) = l;
    };
    // Whether a tile is one that some row sees a part of; its V is looked through for what is not finite.
    auto mixed = [&](uint32_t t) { return t * SLOTS + SLOTS > b.seen && b.seen < b.end; };
    auto watch = [&](uint32_t t, uint32_t stage) {
        if (!isv || t >= b.t1 || !mixed(t)) return;
        bool odd = false;
#pragma unroll
        for (uint32_t i = 0; i < PIECES; i++) odd = odd || odd32(in[i].x) || odd32(in[i].y) || odd32(in[i].z) || odd32(in[i].w);
        if (odd) odd_tile[stage] = t + 1;
    };
    // (A page past the pool: the rows that see its slots are NaN.)
    auto spoil = [&] {
        if (bad)
#pragma unroll
            for (uint32_t i = 0; i < PIECES; i++) in[i] = pg_u32x4{0x7fc00000u, 0x7fc00000u, 0x7fc00000u, 0x7fc00000u};
    };
    auto bad_page = [&](uint32_t t) { return !isv && t < b.t1 && list.bad(t * SLOTS + 16 * half, page); };
    look(b.t0);
    if (threadIdx.x < 2) odd_tile[threadIdx.x] = 0;

    const PgRow row = row_of(p, it, b, wave * 16 + m16);
    bf16x8 q[NB][3];
    {
        f32x4 y[NB][2];
#pragma unroll
        for (int j = 0; j < NB; j++)  // (no branch around them)
#pragma unroll
            for (int e = 0; e < 2; e++) y[j][e] = *(const f32x4*)(p.q + row.at + (32 * j + 8 * g < p.hd ? 32 * j + 8 * g : 0) + 4 * e);
        {
            const __amdgpu_buffer_rsrc_t r = source(b.t0);
#pragma unroll
            for (uint32_t i = 0; i < PIECES; i++) load(r, i);
        }
        bad = bad_page(b.t0);
        look(b.t0 + 1);
#pragma unroll
        for (int j = 0; j < NB; j++) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = row.valid && 32 * j + 8 * g < p.hd ? y[j][e >> 2][e & 3] * p.sc : 0.0f;
            split3(x, q[j]);
        }
    }
    uint32_t kat[NB], vat[NF];
#pragma unroll
    for (int j = 0; j < NB; j++) kat[j] = P::at(m16, 4 * j + g, P::turn_k(m16));
    {
        const uint32_t slot = 4 * g + (m16 >> 2);
#pragma unroll
        for (int f = 0; f < NF; f++) vat[f] = KV + P::at(slot, 2 * f + ((m16 >> 1) & 1), P::turn_v(slot)) + 8 * (m16 & 1);
    }
    f32x4 o[NF];
#pragma unroll
    for (int f = 0; f < NF; f++) o[f] = f32x4{0, 0, 0, 0};
    float ref = -INFINITY, l = 0.0f;
    auto barrier = [] {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
    };
    barrier();  // (odd_tile)
    watch(b.t0, 0);
    spoil();
    {
        const __amdgpu_buffer_rsrc_t r = source(b.t0 + 1);
#pragma unroll
        for (uint32_t i = 0; i < PIECES; i++) {
            put(i, lds);
            load(r, i);
        }
        bad = bad_page(b.t0 + 1);
        look(b.t0 + 2);
    }
    for (uint32_t t = b.t0; t < b.t1; t++) {
        const uint32_t stage = (t - b.t0) & 1, next = 1 - stage, ts = t * SLOTS;
        uint8_t* at = lds + stage * STAGE;
        const bool edge = ts + SLOTS > b.seen;
        barrier();
        if (mixed(t) && odd_tile[stage] == t + 1) {
            // (As in attn_paged_tile16.)
#pragma unroll 1
            for (uint32_t i = 0; i < SLOTS; i++)
#pragma unroll
                for (int f = 0; f < NF; f++) {
                    const half4 v = *(const half4*)(at + KV + (i >> 4) * 3 * P::GRANULE + P::at(i & 15, 2 * f + (g >> 1), P::turn_v(i & 15)) + 8 * (g & 1));
                    if (ts + i < row.vis)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            if ((__builtin_bit_cast(uint16_t, v[e]) & 0x7f80u) == 0x7f80u) o[f][e] = NAN;
                }
            barrier();
            for (uint32_t x = threadIdx.x; x < 2 * 64 * NF; x += 512) {
                uint8_t* v = at + KV + x / (64 * NF) * 3 * P::GRANULE + x % (64 * NF) * 8;
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if ((((const uint16_t*)v)[e] & 0x7f80u) == 0x7f80u)
#pragma unroll
                        for (int z = 0; z < 3; z++) ((uint16_t*)(v + z * P::GRANULE))[e] = 0;
            }
            barrier();
        }
        f32x4 s[2] = {}, s2[2] = {};
#pragma unroll
        for (int j = 0; j < NB; j++) {
            bf16x8 k[2][3];
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int z = 0; z < 3; z++) k[h][z] = *(const bf16x8*)(at + (3 * h + z) * P::GRANULE + kat[j]);
            // (Four sums in turn, so that no MFMA waits for the one before.)
#pragma unroll
            for (int z = 0; z < 6; z++) {
                constexpr int KP[6] = {2, 1, 0, 1, 0, 0}, QP[6] = {0, 1, 2, 0, 1, 0};
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    f32x4& sum = z % 2 ? s[h] : s2[h];
                    sum = mfma_bf16(k[h][KP[z]], q[j][QP[z]], sum);
                }
            }
        }
        bf16x8 w[3];
        s[0] += s2[0];
        s[1] += s2[1];
        if (edge)
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (ts + 16 * (e >> 2) + 4 * g + (e & 3) >= row.vis) s[e >> 2][e & 3] = -INFINITY;
        float f;
        if (raise(s, 1.0f, ref, f)) {
            l *= f;
#pragma unroll
            for (int k = 0; k < NF; k++) o[k] *= f;
        }
        {
            const float base = ref == -INFINITY ? 0.0f : ref;
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                x[e] = exp2_hw(s[e >> 2][e & 3] - base);
                l += x[e];
            }
            split3(x, w);
        }
        const __amdgpu_buffer_rsrc_t after = source(t + 2);
        watch(t + 1, next);
        spoil();
#pragma unroll
        for (int f = 0; f < NF; f += 2) {
            bf16x8 v[2][3];
#pragma unroll
            for (int e = 0; e < 2; e++)
#pragma unroll
                for (int z = 0; z < 3; z++) {
                    const half4 x = read_transposed(at + z * P::GRANULE + vat[f + e]), y = read_transposed(at + (3 + z) * P::GRANULE + vat[f + e]);
                    v[e][z] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
                }
#pragma unroll
            for (int z = 0; z < 6; z++) {
                constexpr int VP[6] = {2, 1, 0, 1, 0, 0}, WP[6] = {0, 1, 2, 0, 1, 0};
#pragma unroll
                for (int e = 0; e < 2; e++) o[f + e] = mfma_bf16(v[e][VP[z]], w[WP[z]], o[f + e]);
            }
            put(f / 2, lds + next * STAGE);  // (the next tile's parts, a share beside each operand)
            load(after, f / 2);
        }
        bad = bad_page(t + 2);
        look(t + 3);
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (!row.valid) return;
    if (b.nchunk > 1) {
        const size_t u = b.unit + wave * b.next;
        f32x4* part = (f32x4*)p.part_o + u * NF * 64 + lane;
#pragma unroll
        for (int f = 0; f < NF; f++) part[64 * f] = o[f];
        if (g == 0) *(float2*)(p.part_ml + 2 * (u * 16 + m16)) = float2{ref, l};
        return;
    }
    const float k = 1.0f / l;
#pragma unroll
    for (int f = 0; f < NF; f++) {
        const uint32_t d = 16 * f + 4 * g;
        if (d < p.hd) *(f32x4*)(p.out + row.at + d) = o[f] * k;
    }
}

template <int NB, int RT>
__global__ __launch_bounds__(RT == 1 ? 512 : 256, 2) void attn_paged_tile16(const PgParams p) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[PG_TILE_LDS<f16, NB>];
    tile16_block<NB, RT>(p, blockIdx.x, lds);
}
template <int NB>
__global__ __launch_bounds__(256, NB > 4 ? 1 : 2) void attn_paged_tile32(const PgParams p) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[PG_TILE_LDS<float, NB>];
    tile32_block<NB>(p, blockIdx.x, lds);
}
template <int NB>
__global__ __launch_bounds__(512, 2) void attn_paged_tile3(const PgParams p) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[PG_TILE3_LDS<NB>];
    tile3_block<NB>(p, blockIdx.x, lds);
}

// A batch of both kinds in one launch: the second kind's blocks first, which take longest and are bound by the
// matrix cores, the first kind's beside and behind them, bound by memory. MIXED: where those start (a
// multiple of 8: their place among the XCDs).
__host__ __device__ __forceinline__ uint32_t mixed_rows(const PgParams& p) { return (p.tblocks * p.nkv + 7) / 8 * 8; }

template <int NB, int RT, bool PK>
__global__ __launch_bounds__(RT == 1 ? 512 : 256, 2) void attn_paged_mixed16(const PgParams p) {
    constexpr int WAVES = RT == 1 ? 8 : 4;
    __shared__ __attribute__((aligned(16))) uint8_t lds[std::max(PG_TILE_LDS<f16, NB>, PG_ROW_LDS<f16, NB, WAVES>)];
    const uint32_t rows = mixed_rows(p);
    if (blockIdx.x >= rows) row_block<f16, NB, PK, WAVES>(p, blockIdx.x - rows, lds);
    else if (blockIdx.x < p.tblocks * p.nkv) tile16_block<NB, RT>(p, blockIdx.x, lds);
}
template <int NB>
__global__ __launch_bounds__(256, NB > 4 ? 1 : 2) void attn_paged_mixed32(const PgParams p) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[std::max(PG_TILE_LDS<float, NB>, PG_ROW_LDS<float, NB, 4>)];
    const uint32_t rows = mixed_rows(p);
    if (blockIdx.x >= rows) row_block<float, NB, false, 4>(p, blockIdx.x - rows, lds);
    else if (blockIdx.x < p.tblocks * p.nkv) tile32_block<NB>(p, blockIdx.x, lds);
}
template <int NB>
__global__ __launch_bounds__(512, 2) void attn_paged_mixed3(const PgParams p) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[std::max(PG_TILE3_LDS<NB>, PG_ROW_LDS<float, NB, 8>)];
    const uint32_t rows = mixed_rows(p);
    if (blockIdx.x >= rows) row_block<float, NB, false, 8>(p, blockIdx.x - rows, lds);
    else if (blockIdx.x < p.tblocks * p.nkv) tile3_block<NB>(p, blockIdx.x, lds);
}

// The chunks of 16 query rows of a list brought together, those that some of the rows see. An operand's columns are
// a wave's (WAVES 1: a workgroup takes fold_share operands), or its chunks' a share for each of WAVES waves;
// states lie as their waves held them. A chunk without a weight left its columns unwritten.
constexpr uint32_t fold_share(int nf) { return nf <= 8 ? nf : nf / 2; }

template <typename KVT, int NB, int WAVES>
__global__ __launch_bounds__(64 * (WAVES == 1 ? fold_share(2 * NB) : WAVES)) void attn_paged_fold(const PgParams p) {
    constexpr int NF = 2 * NB, AHEAD = 8;
    __shared__ f32x4 sum[WAVES][64];
    __shared__ float sr[WAVES][64], sl[WAVES][64];
    const uint32_t lane = threadIdx.x & 63, at_wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), m16 = lane & 15, g = lane >> 4;
    const uint32_t wave = WAVES == 1 ? 0 : at_wave, f = WAVES == 1 ? blockIdx.z * fold_share(NF) + at_wave : blockIdx.z, kvh = blockIdx.y;
    uint32_t which;
    const PgItem it = item_with_arguments<true>(p, false, blockIdx.x, which);
    const bool row = which < p.nrow;
    const uint32_t slots = (row ? 16 : 32) * (sizeof(KVT) == 2 ? 2 : 1), qt = row ? 16 : p.qt;  // of a tile, of a block
    const uint32_t rows = it.rows_seq >> 8, nq = rows * p.G, groups = ((nq - 1) / qt + 1) * (qt / 16);
    const uint32_t chunk = row ? p.chunk : p.tchunk, chunks = ((it.len - 1) / slots) / chunk + 1, group = blockIdx.x - it.fold0, n = 16 * group + m16;
    const uint32_t seen = ((it.len - rows + min(16 * group + 15, nq - 1) / p.G) / slots) / chunk + 1;
    const bool valid = n < nq;
    const size_t u0 = (row ? 0 : (size_t)p.blocks * p.nkv) + (size_t)it.block0 * p.nkv * (qt / 16) + ((size_t)kvh * groups + group) * chunks;
    const float2* ml = (const float2*)p.part_ml + u0 * 16 + m16;
    const f32x4* at = (const f32x4*)p.part_o + (u0 * NF + f) * 64 + lane;
    f32x4 a = {0, 0, 0, 0};
    float R = -INFINITY, L = 0.0f;
    for (uint32_t c0 = wave; c0 < seen; c0 += AHEAD * WAVES) {
        float2 s[AHEAD];
        f32x4 x[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            const uint32_t c = c0 + i * WAVES;
            const bool there = valid && c < seen;
            s[i] = there ? ml[(size_t)c * 16] : float2{-INFINITY, 0.0f};
            x[i] = there ? at[(size_t)c * NF * 64] : f32x4{0, 0, 0, 0};
        }
        float to = R;
#pragma unroll
        for (int i = 0; i < AHEAD; i++) to = fmaxf(to, s[i].x);
        const float ts = to == -INFINITY ? 0.0f : to, w = exp2_hw(R - ts);
        a *= w;
        L *= w;
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            const float e = exp2_hw(s[i].x - ts);
            L += e * s[i].y;
            a += s[i].y == 0.0f ? f32x4{0, 0, 0, 0} : e * x[i];
        }
        R = to;
    }
    if constexpr (WAVES > 1) {
        sr[wave][lane] = R;
        sl[wave][lane] = L;
        sum[wave][lane] = a;
        __syncthreads();
        if (wave > 0) return;
        for (int w = 1; w < WAVES; w++) R = fmaxf(R, sr[w][lane]);
        const float Rs = R == -INFINITY ? 0.0f : R;
        a = f32x4{0, 0, 0, 0};
        L = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; w++) {
            const float e = exp2_hw(sr[w][lane] - Rs);
            L += e * sl[w][lane];
            a += e * sum[w][lane];
        }
    }
    if (!valid) return;
    const float k = 1.0f / L;
    const uint32_t r = n / p.G;
    float* dst = p.out + ((size_t)(it.row0 + r) * p.nh + kvh * p.G + n - r * p.G) * p.hd;
    if (sizeof(KVT) == 2 || qt == 128) {
        const uint32_t d = 16 * f + 4 * g;
        if (d < p.hd) *(f32x4*)(dst + d) = a * k;
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) {
            const uint32_t d = dim_of<KVT, NB>(f, g, i);
            if (d < p.hd) dst[d] = a[i] * k;
        }
    }
}

template <typename KVT, int NB>
void launch_fold(const PgParams& p, uint32_t groups, uint32_t most, hipStream_t s) {
    // A wave alone holds eight chunks' states at once; more chunks are shared out, among few waves where there
    // are many groups (two prompts' pieces beside ten steps: 30 us by eight waves, as their longest list would have
    // it, 14 by two). 25 MB of states of such pieces and their results take 9 us, of which stores of 4
    // bytes had cost 3.
    const dim3 grid(groups, p.nkv, 2 * NB);
    constexpr uint32_t share = fold_share(2 * NB);
    if (most <= 8) hipLaunchKernelGGL((attn_paged_fold<KVT, NB, 1>), dim3(groups, p.nkv, 2 * NB / share), dim3(64 * share), 0, s, p);
    else if (most <= 16 || groups >= 64) hipLaunchKernelGGL((attn_paged_fold<KVT, NB, 2>), grid, dim3(128), 0, s, p);
    else hipLaunchKernelGGL((attn_paged_fold<KVT, NB, 8>), grid, dim3(512), 0, s, p);
}

template <int NB>
void launch_tile16(const PgParams& p, hipStream_t s) {
    const dim3 grid(p.tblocks * p.nkv);
    if constexpr (NB <= 4) {
        if (p.qt == 128) {
            hipLaunchKernelGGL((attn_paged_tile16<NB, 2>), grid, dim3(256), 0, s, p);
            return;
        }
    }
    hipLaunchKernelGGL((attn_paged_tile16<NB, 1>), grid, dim3(512), 0, s, p);
}
template <int NB>
void launch_tile32(const PgParams& p, hipStream_t s) {
    const dim3 grid(p.tblocks * p.nkv);
    if constexpr (NB <= 4) {
        if (p.qt == 128) {
            hipLaunchKernelGGL((attn_paged_tile3<NB>), grid, dim3(512), 0, s, p);
            return;
        }
    }
    hipLaunchKernelGGL((attn_paged_tile32<NB>), grid, dim3(256), 0, s, p);
}
template <int NB>
void launch_mixed(const PgParams& p, bool f16_cache, hipStream_t s) {
    const dim3 grid(mixed_rows(p) + (p.blocks + 7) / 8 * 8 * p.nkv);
    if constexpr (NB <= 4) {
        const bool few = pg_few(p);
        if (!f16_cache && p.qt == 128) hipLaunchKernelGGL((attn_paged_mixed3<NB>), grid, dim3(512), 0, s, p);
        else if (!f16_cache) hipLaunchKernelGGL((attn_paged_mixed32<NB>), grid, dim3(256), 0, s, p);
        else if (p.qt == 128 && few) hipLaunchKernelGGL((attn_paged_mixed16<NB, 2, true>), grid, dim3(256), 0, s, p);
        else if (p.qt == 128) hipLaunchKernelGGL((attn_paged_mixed16<NB, 2, false>), grid, dim3(256), 0, s, p);
        else if (few) hipLaunchKernelGGL((attn_paged_mixed16<NB, 1, true>), grid, dim3(512), 0, s, p);
        else hipLaunchKernelGGL((attn_paged_mixed16<NB, 1, false>), grid, dim3(512), 0, s, p);
    } else {
        hipLaunchKernelGGL((attn_paged_mixed32<NB>), grid, dim3(256), 0, s, p);
    }
}

uint32_t ceil_div(uint64_t a, uint64_t b) { return (uint32_t)((a + b - 1) / b); }

// What a launch over p's items in chunks of p.chunk and p.tchunk tiles takes: the blocks' places, the
// states, and the groups of the fold (items whose lists are whole have none).
struct PgPlan {
    uint64_t states = 0;  // groups of 16 query rows
    uint32_t groups = 0, most = 1;
};
PgPlan place(PgParams& p, bool f16_cache) {
    PgPlan plan;
    p.blocks = p.tblocks = 0;
    for (uint32_t i = 0; i < p.nitems; i++) {
        PgItem& it = p.items[i];
        const bool row = i < p.nrow;
        const uint32_t nq = (it.rows_seq >> 8) * p.G, chunks = (it.len - 1) / (row ? pg_row_tile(f16_cache) : pg_tile(f16_cache)) / (row ? p.chunk : p.tchunk) + 1;
        uint32_t& blocks = row ? p.blocks : p.tblocks;
        it.block0 = blocks;
        it.fold0 = plan.groups;
        blocks += (row ? 1 : ceil_div(nq, p.qt)) * chunks;
        if (chunks > 1) plan.groups += ceil_div(nq, 16);
        plan.most = std::max(plan.most, chunks);
    }
    plan.states = ((uint64_t)p.blocks + (uint64_t)p.tblocks * (p.qt / 16)) * p.nkv;
    return plan;
}

bool reserve(PgParams& p, const PgPlan& plan, Workspace& ws) {
    const uint32_t hd = p.hd;  // (states are those of the kernel's head, at most the next power of two)
    const bool had = ws.reserve_if(plan.states * 16, hd <= 32 ? 32 : hd <= 64 ? 64 : hd <= 128 ? 128 : 256);
    p.part_o = ws.o;
    p.part_ml = ws.ml;
    return had;
}

constexpr uint32_t WHOLE = 0x40000000u;  // tiles: no list has as many

// K and V of the items of at most 16 query rows.
uint64_t row_bytes(const PgParams& p, bool f16_cache) {
    uint64_t slots = 0;
    for (uint32_t i = 0; i < p.nrow; i++) slots += p.items[i].len;
    return slots * p.nkv * p.hd * (f16_cache ? 4 : 8);
}

// Items of at most 16 query rows: the chunks. Whether they are brief: lists that eight waves take in a few
// tiles each are not cut (no second launch).
bool cut_rows(PgParams& p, bool f16_cache) {
    const uint32_t slots = pg_row_tile(f16_cache);
    uint64_t total = 0, most = 0;
    for (uint32_t i = 0; i < p.nrow; i++) {
        const uint64_t tiles = (p.items[i].len - 1) / slots + 1;
        total += tiles;
        most = std::max(most, tiles);
    }
    p.chunk = WHOLE;
    if (most <= 20) return true;
    // Chunks of whole rounds of the waves, as short as leaves every workgroup a place at once, 512; beside blocks
    // of the second kind, which take most places, one for every 200 KB, 192 to 512 (29 steps of up to 6000 slots
    // beside a piece of a prompt, 28 x 4 heads of 128: 64 us by 512, 87 by 128; two pieces and ten steps 78 by
    // 192, 82 by 512; verify passes of 1 to 6 rows before 5000 slots, 64 x 8 heads: 24.6, 27.0).
    const uint32_t groups = p.nrow == p.nitems ? 512 : (uint32_t)std::min<uint64_t>(512, std::max<uint64_t>(192, row_bytes(p, f16_cache) / 200000));
    p.chunk = std::max<uint32_t>(4, ceil_div(ceil_div(total * p.nkv, groups), 4) * 4);
    auto blocks = [&] {
        uint64_t n = 0;
        for (uint32_t i = 0; i < p.nrow; i++) n += (p.items[i].len - 1) / slots / p.chunk + 1;
        return n * p.nkv;
    };
    while (p.chunk < most && blocks() > groups) p.chunk += std::max(4u, p.chunk / 16 / 4 * 4);
    return false;
}

// What a launch over the items of more in blocks of qt query rows takes, and in which chunks. It is counted out: a
// KV head's share of the CUs takes its blocks in their order, each the place that is free first, one or two a
// CU as LDS has it. A block's start (arguments, pages, q, the first tile) takes START us, a tile `paired` us
// beside another block and `alone` of that without one; the fold FOLD us and its states' bytes. (Within 5%
// of what launches in any chunks were measured to take: 600 rows before 2000 slots, 32 x 8 heads of 128 in
// f16, 62 to 104 us; the pieces of two prompts 77 to 115; 777 rows in f32 75 to 96. The chunks that it picks:
// 63, 78 and 76.)
struct PgCut {
    float us;
    uint32_t chunk;
};
PgCut cut(const PgParams& p, bool f16_cache, uint32_t qt, uint32_t longest, float limit) {
    constexpr uint32_t CUS = 256, TIMES = 512, NONE = 0xffff;
    constexpr float START = 6.5f, FOLD = 5.5f;
    const uint32_t slots = pg_tile(f16_cache);
    const bool whole_cu = !f16_cache && qt == 128 && p.hd > 96;
    const float paired = f16_cache ? (qt == 128 ? 0.36f + 0.02f * p.hd : 0.28f + 0.015f * p.hd) : qt == 128 ? (whole_cu ? 0.0195f : 0.039f) * p.hd : 0.027f * p.hd;
    const float alone = f16_cache ? (qt == 128 ? 0.8f : 0.65f) : 0.7f;
    uint32_t tiles[4 * CUS], units = 0;  // of a KV head's query blocks
    uint64_t sum = 0, all = 0;
    for (uint32_t i = p.nrow; i < p.nitems; i++) {
        const PgItem& it = p.items[i];
        const uint32_t rows = it.rows_seq >> 8, nqt = ceil_div(rows * p.G, qt);
        all += (uint64_t)nqt * ((it.len - rows / 2 - 1) / slots + 1);
        if ((uint64_t)(units + nqt) * p.nkv >= 4 * CUS) units = 4 * CUS;
        if (units == 4 * CUS) continue;
        for (uint32_t x = nqt; x-- > 0; sum += tiles[units++]) tiles[units] = (it.len - rows + std::min(((x + 1) * qt - 1) / p.G, rows - 1)) / slots + 1;
    }
    const uint32_t cus = std::max(1u, CUS / p.nkv), places = whole_cu ? cus : 2 * cus;
    if (units == 4 * CUS) return {(float)all * paired / places + START, WHOLE};  // (every CU has several: nothing to be had)
    const float evenly = (START * units + (float)sum * paired) / places, unit = (START + longest * paired + evenly) / (TIMES / 2);  // of the count
    if (0.7f * evenly > limit) return {limit, WHOLE};
    const float start = START / unit + 0.5f, each = paired / unit, state = (float)p.nkv * qt * p.hd * 8 / 6.4e6f;
    auto time = [&](uint32_t chunk) {
        uint16_t first[TIMES], next[2 * CUS], ends[2 * CUS];  // places that are free at a time, one after another
        std::fill(first, first + TIMES, NONE);
        std::fill(ends, ends + places, 0);
        for (uint32_t x = 0; x < places; x++) next[x] = (uint16_t)(x + 1);
        next[places - 1] = NONE;
        first[0] = 0;
        uint32_t now = 0, states = 0, at = 0;
        for (uint32_t i = p.nrow; i < p.nitems; i++) {
            const uint32_t nqt = ceil_div((p.items[i].rows_seq >> 8) * p.G, qt), chunks = (tiles[at] - 1) / chunk + 1;
            if (chunks > 1) states += nqt * chunks;
            for (uint32_t c = 0; c < chunks; c++)
                for (uint32_t x = at; x < at + nqt && tiles[x] > c * chunk; x++) {
                    while (first[now] == NONE) now++;
                    const uint32_t place = first[now];
                    first[now] = next[place];
                    const uint32_t to = std::min(now + (uint32_t)(start + std::min(chunk, tiles[x] - c * chunk) * each), TIMES - 1);
                    ends[place] = (uint16_t)to;
                    next[place] = first[to];
                    first[to] = (uint16_t)place;
                }
            at += nqt;
        }
        float last = 0.0f;
        for (uint32_t x = 0; x < cus; x++) {
            const int a = ends[x], b = whole_cu ? a : ends[x + cus];
            last = std::max(last, std::min(a, b) + (float)std::abs(a - b) * alone);
        }
        return last * unit + (states ? FOLD + states * state : 0.0f);
    };
    PgCut best = {time(longest), WHOLE};
    for (uint32_t chunk = longest; chunk > 2;) {
        chunk = std::min(chunk - 1, chunk * 27 / 32);
        const uint32_t many = units * ceil_div(longest, chunk);  // (the count itself takes the host's time)
        if (many > 320 || many * p.nkv > 8 * CUS || 0.7f * evenly + FOLD + (float)sum / chunk * state > best.us) break;
        const float t = time(chunk);
        if (t < best.us) best = {t, chunk};
    }
    return best;
}

// Items of more: query rows a block, and the chunks. Where most items have more than 64 query rows blocks of 128,
// whose tiles are read half as often (and f32 heads of up to 128 dims run in bf16 parts, the few smaller items among
// them too); f16 heads in blocks of 64 where those end sooner, there being few blocks
// (494 rows, 32 x 8 heads of 128: 18 us, 27 by 128; before 1500 slots, 28 x 4 heads: 45, 48; 600 before
// 2000, 32 x 8: 78, 63).
void cut_tiles(PgParams& p, bool f16_cache) {
    const uint32_t slots = pg_tile(f16_cache);
    std::sort(p.items + p.nrow, p.items + p.nitems, [](const PgItem& a, const PgItem& b) { return a.len > b.len; });
    uint32_t few = 0, many = 0, longest = 0;  // items of at most 64 query rows, of more; a list's tiles
    for (uint32_t i = p.nrow; i < p.nitems; i++) {
        ((uint64_t)(p.items[i].rows_seq >> 8) * p.G <= 64 ? few : many)++;
        longest = std::max(longest, (p.items[i].len - 1) / slots + 1);
    }
    p.qt = p.hd <= 128 && many >= few ? 128 : 64;
    PgCut best = cut(p, f16_cache, p.qt, longest, INFINITY);
    // (Beside longer work of the first kind, at 5 MB a us, blocks of 128 leave it more of LDS: 40 steps of up to 3000
    // slots and 100 rows, 32 x 8 heads of 128, 73 us, 79 by 64.)
    if (f16_cache && p.qt == 128 && row_bytes(p, f16_cache) / 5e6f < best.us) {
        const PgCut other = cut(p, f16_cache, 64, longest, best.us);
        if (other.us < best.us) best = other, p.qt = 64;
    }
    p.tchunk = best.chunk;
}

hipError_t run(PgParams& p, bool f16_cache, Workspace& ws, hipStream_t s) {
    p.qt = 64;
    p.chunk = p.tchunk = WHOLE;
    const bool rows = p.nrow > 0, tiles = p.nrow < p.nitems;
    if (tiles) cut_tiles(p, f16_cache);
    const bool brief = rows && cut_rows(p, f16_cache);
    PgPlan plan = place(p, f16_cache);
    if (plan.groups && !reserve(p, plan, ws)) {  // whole lists
        p.chunk = p.tchunk = WHOLE;
        plan = place(p, f16_cache);
    }
    if (rows && tiles && (!f16_cache || p.hd <= 128)) {
        paged_mixed_launch(p, f16_cache, s);
    } else {
        if (rows) paged_rows_launch(p, f16_cache, brief, s);
        if (tiles) paged_tiles_launch(p, f16_cache, s);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || !plan.groups) return e;
    paged_fold_launch(p, f16_cache, plan.groups, plan.most, s);
    return hipGetLastError();
}

}  // namespace

void paged_tiles_launch(const PgParams& p, bool f16_cache, hipStream_t s) {
#define PG_TILE(NB) (f16_cache ? launch_tile16<NB>(p, s) : launch_tile32<NB>(p, s))
    PG_BY_DIM(p.hd, PG_TILE)
#undef PG_TILE
}

void paged_mixed_launch(const PgParams& p, bool f16_cache, hipStream_t s) {
#define PG_MIXED(NB) launch_mixed<NB>(p, f16_cache, s)
    PG_BY_DIM(p.hd, PG_MIXED)
#undef PG_MIXED
}

void paged_fold_launch(const PgParams& p, bool f16_cache, uint32_t groups, uint32_t most, hipStream_t s) {
#define PG_FOLD(NB) (f16_cache ? launch_fold<f16, NB>(p, groups, most, s) : launch_fold<float, NB>(p, groups, most, s))
    PG_BY_DIM(p.hd, PG_FOLD)
#undef PG_FOLD
}

hipError_t paged_attention(const PagedCall& a, Workspace& ws, hipStream_t s) {
    const bool f16_cache = a.kv_type == 1;
    PgParams base{};
    base.q = a.q;
    base.kc = (const uint8_t*)a.kc;
    base.vc = (const uint8_t*)a.vc;
    base.out = a.out;
    base.pages = a.pages.table;
    base.page_stride = a.pages.stride;
    base.page_shift = a.pages.shift;
    base.npages = a.pages.npages;
    base.nh = a.nh;
    base.nkv = a.nkv;
    base.hd = a.hd;
    base.G = a.nh / a.nkv;
    base.sc = a.scale * LOG2E;
    // Sequences with rows, the first kind first, as many as a launch takes at a time.
    uint32_t next = 0;
    while (next < a.pages.nseq) {
        PgParams p = base;
        uint32_t end = next, n = 0;
        for (; end < a.pages.nseq && n < PG_ITEMS; end++) n += a.pages.starts[end + 1] > a.pages.starts[end];
        for (int many = 0; many < 2; many++) {
            if (many) p.nrow = p.nitems;
            for (uint32_t i = next; i < end; i++) {
                const uint32_t rows = a.pages.starts[i + 1] - a.pages.starts[i];
                if (rows == 0 || ((uint64_t)rows * base.G > 16) != (many == 1)) continue;
                p.items[p.nitems++] = PgItem{a.pages.starts[i], a.pages.lens[i], rows << 8 | i, 0, 0};
            }
        }
        next = end;
        if (p.nitems == 0) continue;
        const hipError_t e = run(p, f16_cache, ws, s);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace bchip
