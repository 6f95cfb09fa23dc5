// Attention over a cache in pages (paged.hpp) of at most 16 query rows a KV head (rows x the heads
// that share it): decode steps of several sequences in one launch, short verify passes. The kernels are
// attn_paged_row, and beside the blocks of more query rows attn_paged_mixed16, 3 and 32.
//
// Mathematics. f16 caches: K and V are f16 operands as they lie, q and the softmax weights two f16
// each (parts.hpp). f32 caches: f32 products and sums on the f32 matrix cores. So a result is as near
// as f32 arithmetic comes to the formula over the stored values.
//
// Layout. Scores are S^T = K q^T, 16 slots x 16 query rows an MFMA, whose result leaves lane (n, g) with
// slots 4g .. 4g + 3 of query row n: the B operand of O^T = V^T P^T with the slots numbered that way, so
// the weights never leave their lane. f16: V comes out of LDS transposed; up to eight query rows put
// q's and the weights' two parts side by side in the MFMA's columns (PK), half the matrix work. f32: a
// lane's 16 bytes of V are four operands' columns.
//
// A workgroup takes a chunk of a list, each of its waves every WAVES'th tile of it alone, K and V on
// their way into the wave's own LDS while the tile before is computed: K's next tile is asked for once
// this one's is in registers, V's likewise, so both are always on their way and a wave needs one tile
// of LDS. The waves' states meet in LDS, chunks in attn_paged_fold. Blocks eight apart (one XCD) take
// the KV heads of one chunk.
//
// Bound by the bytes of K and V: 16 steps at up to 24001 slots, 32 x 8 heads of 128 in f16, take 137 us and
// the fold 4.8 (5.07 TB/s together; a large copy reaches 5.15), 16 at up to 8000 in f32 95 us (5.05). A list of
// 400 slots takes 6.5 us, the latency of arguments, page number, first tile and the states' way through LDS.
#pragma once

#include "paged.hpp"
#include "parts.hpp"

namespace bchip {

// Bytes of LDS of a workgroup: each wave's K and V tile, the states' references and sums.
template <typename KVT, int NB, int WAVES>
constexpr uint32_t PG_ROW_LDS = WAVES * 2 * (sizeof(KVT) == 2 ? 2 : 1) * PgTile<KVT, NB>::GRANULE + 2 * WAVES * 64 * 4;

// Block `id` of the items of at most 16 query rows. lds: PG_ROW_LDS bytes, 16-byte aligned.
template <typename KVT, int NB, bool PK, int WAVES>
__device__ __forceinline__ void row_block(const PgParams& p, uint32_t id, uint8_t* lds) {
    using T = PgTile<KVT, NB>;
    constexpr bool F16 = sizeof(KVT) == 2;
    constexpr int HD = 32 * NB, NF = 2 * NB, NG = F16 ? 2 : 1, LOADS = NG * T::LOADS, NJ = T::UNITS / 4;
    constexpr uint32_t SLOTS = 16 * NG;
    constexpr uint32_t TILES = WAVES * 2 * NG * T::GRANULE;
    uint8_t(*sh)[2][NG * T::GRANULE] = (uint8_t(*)[2][NG * T::GRANULE])lds;
    float(*sr)[64] = (float(*)[64])(lds + TILES), (*sl)[64] = (float(*)[64])(lds + TILES + WAVES * 64 * 4);
    static_assert(sizeof(f32x4) * 4 * NF * 64 <= TILES, "the waves' states");
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t m16 = lane & 15, g = lane >> 4;
    const uint32_t block = (id / (8 * p.nkv)) * 8 + (id & 7), kvh = (id >> 3) % p.nkv;
    uint32_t which;
    const PgItem it = item_with_arguments<false>(p, true, block, which);
    if (block >= p.blocks) return;
    const uint32_t rows = it.rows_seq >> 8, nq = rows * p.G, seen = it.len - rows + 1;  // slots every row sees
    const PgList list = list_of(p, it, kvh, T::ES);
    const uint32_t all = (it.len - 1) / SLOTS + 1, chunk = block - it.block0, nchunk = (all - 1) / p.chunk + 1;
    const uint32_t first = chunk * p.chunk, tiles = min(p.chunk, all - first);

    // This wave's tiles are first + wave, + WAVES, ...; the one on its way, and the pages of the one after.
    uint8_t *kt = sh[wave][0], *vt = sh[wave][1];
    const uint32_t kl = (uint32_t)(uintptr_t)(pg_lds*)kt, vl = (uint32_t)(uintptr_t)(pg_lds*)vt;
    uint32_t kfrom[T::LOADS], vfrom[T::LOADS], page[NG], bad = 0;
#pragma unroll
    for (int i = 0; i < T::LOADS; i++) {
        kfrom[i] = T::template from<false>(i, lane, list.row_bytes, p.hd * T::ES);
        vfrom[i] = T::template from<true>(i, lane, list.row_bytes, p.hd * T::ES);
    }
    auto look = [&](uint32_t t) {
#pragma unroll
        for (int h = 0; h < NG; h++) page[h] = list.page((first + min(t, tiles)) * SLOTS + 16 * h);
    };
    auto fetch = [&](const uint8_t* cache, const uint32_t (&from)[T::LOADS], uint32_t to, uint32_t t) {
#pragma unroll
        for (int h = 0; h < NG; h++) {
            const pg_u32x4 r = list.granule(cache, t < tiles ? (first + t) * SLOTS + 16 * h : list.end, page[h]);
#pragma unroll
            for (int i = 0; i < T::LOADS; i++) load_lds(r, from[i], to, h * T::GRANULE + 1024 * i);
        }
    };
    look(wave);

    // q's operands.
    const uint32_t n = PK ? (m16 & 7) : m16, r = (n * (65536 / p.G + 1)) >> 16;  // n / G
    const bool valid = n < nq;
    const uint32_t row = it.row0 + (valid ? r : 0), head = kvh * p.G + (valid ? n - r * p.G : 0);
    const uint32_t vis = valid ? seen + r : list.end;  // slots this lane's row sees
    const size_t qrow = ((size_t)row * p.nh + head) * p.hd;
    f32x4 x[NJ][F16 ? 2 : 1];
    auto dim = [&](int j) { return HD / NJ * j + HD / NJ / 4 * g; };
#pragma unroll
    for (int j = 0; j < NJ; j++)  // (no branch around them)
#pragma unroll
        for (int e = 0; e < (F16 ? 2 : 1); e++) x[j][e] = *(const f32x4*)(p.q + qrow + (dim(j) < p.hd ? dim(j) : 0) + 4 * e);
    // They are waited for here, beside the pages: behind the tile's loads, which the compiler does not
    // count, its wait for them would be one for those too.
#pragma unroll
    for (int j = 0; j < NJ; j++)
#pragma unroll
        for (int e = 0; e < (F16 ? 2 : 1); e++) asm volatile("" : "+v"(x[j][e]));
    fetch(p.kc, kfrom, kl, wave);
    fetch(p.vc, vfrom, vl, wave);
#pragma unroll
    for (int h = 0; h < NG; h++) bad |= list.bad((first + wave) * SLOTS + 16 * h, page[h]) ? 1u << h : 0;
    look(wave + WAVES);
#pragma unroll
    for (int j = 0; j < NJ; j++)
#pragma unroll
        for (int e = 0; e < (F16 ? 2 : 1); e++)
            if (!valid || dim(j) >= p.hd) x[j][e] = f32x4{0, 0, 0, 0};
    float c = 1.0f;
    const float keep = PK && m16 >= 8 ? 1.0f : 0.0f;
    half8 qa[F16 ? NB : 1], qb[F16 && !PK ? NB : 1];
    if constexpr (F16) {
        float top = 0.0f, k;
        float y[NB][8];
#pragma unroll
        for (int j = 0; j < NB; j++) {
#pragma unroll
            for (int e = 0; e < 8; e++) y[j][e] = x[j][e >> 2][e & 3];
            top = q_top(y[j], top);
        }
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        q_scale(top, p.sc, k, c);
#pragma unroll
        for (int j = 0; j < NB; j++) {
            half8 hi, lo;
            q_parts(y[j], k, hi, lo);
            if constexpr (PK) {
                qa[j] = m16 < 8 ? hi : lo;
            } else {
                qa[j] = hi;
                qb[j] = lo;
            }
        }
    }
    // Where this lane's operands lie in a granule.
    uint32_t kat[NJ], vat[F16 ? NF : 1];
#pragma unroll
    for (int j = 0; j < NJ; j++) kat[j] = T::at(m16, 4 * j + g, T::turn_k(m16));
    if constexpr (F16) {
        const uint32_t slot = 4 * g + (m16 >> 2);
#pragma unroll
        for (int f = 0; f < NF; f++) vat[f] = T::at(slot, 2 * f + ((m16 >> 1) & 1), T::turn_v(slot)) + 8 * (m16 & 1);
    }

    f32x4 o[NF];
#pragma unroll
    for (int f = 0; f < NF; f++) o[f] = f32x4{0, 0, 0, 0};
    float ref = -INFINITY, l = 0.0f;

    for (uint32_t t = wave; t < tiles; t += WAVES) {
        const uint32_t ts = (first + t) * SLOTS;
        wait_loads<LOADS>();  // K's (V's may be on their way)
        f32x4 s[NG];
        if constexpr (F16) {
            half8 kf[NG][NB];
#pragma unroll
            for (int h = 0; h < NG; h++)
#pragma unroll
                for (int j = 0; j < NB; j++) kf[h][j] = *(const half8*)(kt + h * T::GRANULE + kat[j]);
            wait_lds();
            fetch(p.kc, kfrom, kl, t + WAVES);
            f32x4 s2[NG];
#pragma unroll
            for (int h = 0; h < NG; h++) s[h] = s2[h] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < NB; j++)
#pragma unroll
                for (int h = 0; h < NG; h++) {
                    s[h] = mfma16(kf[h][j], qa[j], s[h]);
                    if constexpr (!PK) s2[h] = mfma16(kf[h][j], qb[j], s2[h]);
                }
#pragma unroll
            for (int h = 0; h < NG; h++)
#pragma unroll
                for (int i = 0; i < 4; i++) s[h][i] += PK ? ror8(s[h][i]) : s2[h][i];
        } else {
            f32x4 kf[NJ], a[4] = {};
#pragma unroll
            for (int j = 0; j < NJ; j++) kf[j] = *(const f32x4*)(kt + kat[j]);
            wait_lds();
            fetch(p.kc, kfrom, kl, t + WAVES);
#pragma unroll
            for (int j = 0; j < NJ; j++)
#pragma unroll
                for (int e = 0; e < 4; e++) a[e] = mfma_f32(kf[j][e], x[j][0][e], a[e]);
#pragma unroll
            for (int i = 0; i < 4; i++) s[0][i] = ((a[0][i] + a[1][i]) + (a[2][i] + a[3][i])) * p.sc;
        }
        if (bad)  // a page past the pool: the rows that see its slots are NaN
#pragma unroll
            for (int h = 0; h < NG; h++)
                if (bad >> h & 1) s[h] = f32x4{NAN, NAN, NAN, NAN};
        // A tile that some row does not see whole: unseen slots' scores become -inf.
        const bool edge = ts + SLOTS > seen;
        if (edge)
#pragma unroll
            for (int h = 0; h < NG; h++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (ts + 16 * h + 4 * g + i >= vis) s[h][i] = -INFINITY;
        float f;
        if (raise(s, c, ref, f)) {
            l *= f;
#pragma unroll
            for (int i = 0; i < NF; i++) o[i] *= f;
        }
        half8 ph, pl;
        if constexpr (F16) {
            weights<PK>(s, c, ref, keep, l, ph, pl);
        } else {
            const float base = ref == -INFINITY ? 0.0f : ref;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                s[0][i] = exp2_hw(s[0][i] - base);
                l += s[0][i];
            }
        }
        wait_loads<LOADS>();  // V's (K's next tile is on its way)
        // An infinity or a NaN in V reaches the rows that see its slot and, its weight being 0, must not
        // reach the others.
        const bool mixed = edge && rows > 1;
        if constexpr (F16) {
            half8 vf[NF];
#pragma unroll
            for (int k = 0; k < NF; k++) {
                const half4 a = read_transposed(vt + vat[k]), b = read_transposed(vt + T::GRANULE + vat[k]);
                vf[k] = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
            }
            wait_lds();
            if (mixed) {
                bool odd = false;
#pragma unroll
                for (int k = 0; k < NF; k++) {
                    pg_u32x4 w = __builtin_bit_cast(pg_u32x4, vf[k]);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        odd |= odd16(w[e]);
                        if ((w[e] & 0x7c00u) == 0x7c00u) w[e] &= 0xffff0000u;
                        if ((w[e] & 0x7c000000u) == 0x7c000000u) w[e] &= 0xffffu;
                    }
                    vf[k] = __builtin_bit_cast(half8, w);
                }
                if (__any(odd)) {
                    for (uint32_t i = 0; i < SLOTS; i++) {
                        const uint32_t y = i & 15;
#pragma unroll
                        for (int k = 0; k < NF; k++) {
                            const half4 v = *(const half4*)(vt + (i >> 4) * T::GRANULE + T::at(y, 2 * k + (g >> 1), T::turn_v(y)) + 8 * (g & 1));
                            if (ts + i < vis)
#pragma unroll
                                for (int e = 0; e < 4; e++)
                                    if (odd16(__builtin_bit_cast(uint16_t, v[e]))) o[k][e] = NAN;
                        }
                    }
                    wait_lds();
                }
            }
            fetch(p.vc, vfrom, vl, t + WAVES);
#pragma unroll
            for (int k = 0; k < NF; k++) o[k] = mfma16(vf[k], ph, o[k]);
            if constexpr (!PK) {
#pragma unroll
                for (int k = 0; k < NF; k++) o[k] = mfma16(vf[k], pl, o[k]);
            }
        } else {
            constexpr int NS = NB / 2, TAIL = NB % 2;
            f32x4 vf[4][NS > 0 ? NS : 1];
            f32x2 vs[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint8_t* at = vt + (4 * g + i) * T::PITCH;
#pragma unroll
                for (int z = 0; z < NS; z++) vf[i][z] = *(const f32x4*)(at + 256 * z + 16 * m16);
                if constexpr (TAIL) vs[i] = *(const f32x2*)(at + 256 * NS + 8 * m16);
            }
            wait_lds();
            if (mixed) {
                bool odd = false;
#pragma unroll
                for (int i = 0; i < 4; i++) {
#pragma unroll
                    for (int z = 0; z < NS; z++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            if (odd32(__float_as_uint(vf[i][z][e]))) vf[i][z][e] = 0.0f, odd = true;
                    if constexpr (TAIL)
#pragma unroll
                        for (int e = 0; e < 2; e++)
                            if (odd32(__float_as_uint(vs[i][e]))) vs[i][e] = 0.0f, odd = true;
                }
                if (__any(odd)) {
                    for (uint32_t i = 0; i < SLOTS && ts + i < vis; i++)
#pragma unroll
                        for (int k = 0; k < NF; k++)
#pragma unroll
                            for (int e = 0; e < 4; e++)
                                if (odd32(*(const uint32_t*)(vt + i * T::PITCH + 4 * dim_of<KVT, NB>(k, g, e)))) o[k][e] = NAN;
                    wait_lds();
                }
            }
            fetch(p.vc, vfrom, vl, t + WAVES);
#pragma unroll
            for (int i = 0; i < 4; i++) {
#pragma unroll
                for (int z = 0; z < NS; z++)
#pragma unroll
                    for (int e = 0; e < 4; e++) o[4 * z + e] = mfma_f32(vf[i][z][e], s[0][i], o[4 * z + e]);
                if constexpr (TAIL)
#pragma unroll
                    for (int e = 0; e < 2; e++) o[4 * NS + e] = mfma_f32(vs[i][e], s[0][i], o[4 * NS + e]);
            }
        }
        bad = 0;
#pragma unroll
        for (int h = 0; h < NG; h++) bad |= t + WAVES < tiles && list.bad((first + t + WAVES) * SLOTS + 16 * h, page[h]) ? 1u << h : 0;
        look(t + 2 * WAVES);
    }
    wait_loads<0>();  // (zeros behind the last tile, into LDS that the states are to take)

    // The waves' states, lane by lane: the upper half of more than four to the lower, then each of
    // four waves brings some of the columns together.
    f32x4(*so)[NF][64] = (f32x4(*)[NF][64])lds;
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if constexpr (PK) {
#pragma unroll
        for (int f = 0; f < NF; f++)
#pragma unroll
            for (int i = 0; i < 4; i++) o[f][i] += ror8(o[f][i]);
    }
#pragma unroll
    for (uint32_t half = WAVES / 2; half >= 4; half /= 2) {
        __syncthreads();
        if (wave >= half && wave < 2 * half) {
            sr[wave][lane] = ref;
            sl[wave][lane] = l;
#pragma unroll
            for (int f = 0; f < NF; f++) so[wave - half][f][lane] = o[f];
        }
        __syncthreads();
        if (wave < half) {
            const float other = sr[wave + half][lane], to = fmaxf(ref, other), ts = to == -INFINITY ? 0.0f : to;
            const float a = exp2_hw(ref - ts), e = exp2_hw(other - ts);
            l = l * a + sl[wave + half][lane] * e;
#pragma unroll
            for (int f = 0; f < NF; f++) o[f] = o[f] * a + so[wave][f][lane] * e;
            ref = to;
        }
    }
    __syncthreads();
    if (wave < 4) {
        sr[wave][lane] = ref;
        sl[wave][lane] = l;
#pragma unroll
        for (int f = 0; f < NF; f++) so[wave][f][lane] = o[f];
    }
    __syncthreads();
    if (wave >= 4 || !valid || (PK && m16 >= 8)) return;
    float a[4], L = 0.0f;
    const float R = fmaxf(fmaxf(sr[0][lane], sr[1][lane]), fmaxf(sr[2][lane], sr[3][lane])), Rs = R == -INFINITY ? 0.0f : R;
#pragma unroll
    for (int w = 0; w < 4; w++) {
        a[w] = exp2_hw(sr[w][lane] - Rs);
        L += sl[w][lane] * a[w];
    }
    const size_t unit = (size_t)it.block0 * p.nkv + kvh * nchunk + chunk;
    const float inv = nchunk > 1 ? 1.0f : 1.0f / L;
    if (nchunk > 1 && wave == 0 && g == 0) *(float2*)(p.part_ml + 2 * (unit * 16 + n)) = float2{R, L};
    for (uint32_t f = wave; f < NF; f += 4) {
        f32x4 v = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < 4; w++) v += so[w][f][lane] * a[w];
        v *= inv;
        if (nchunk > 1) {
            *(f32x4*)(p.part_o + ((unit * NF + f) * 64 + lane) * 4) = v;
        } else if constexpr (F16) {
            if (16 * f + 4 * g < p.hd) *(f32x4*)(p.out + qrow + 16 * f + 4 * g) = v;
        } else {
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) {
                const uint32_t d = dim_of<KVT, NB>(f, g, i);
                if (d < p.hd) p.out[qrow + d] = v[i];
            }
        }
    }
}

}  // namespace bchip
