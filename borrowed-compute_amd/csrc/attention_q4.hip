// Attention over caches in 4 bits (q4.hpp): out[r][h] = softmax(scale q k^T) v over the slots
// that row r sees, for decode steps, verify passes, trees, prompts and ragged pools.
//
// Mathematics. A cached value (code - 8) d is exactly an f16 (q4.hpp), so K and V feed the f16
// matrix cores as they are. q (times scale log2 e, brought to 2^13 .. 2^14 by a power of two of
// its row) and the softmax weights go in as two f16 each, the rounded value and the rest: 22
// bits, every product exact, sums in f32. So a result is as near as f32 arithmetic comes to the
// formula, at twice the matrix work of f16 operands.
//
// Layout. Scores are S^T = K q^T, 16 slots x 16 query rows (rows x the heads that share a KV
// head) an MFMA. Its result leaves lane (n, g) with slots 4g .. 4g + 3 of query row n, which is
// how the B operand of O^T = V^T P^T wants the weights if the slots of two such blocks are
// numbered that way: the weights never leave their lane. A lane takes eight of those slots' codes
// of V as words of the same columns, so pairs of slots unpack side by side and a lane's eight
// columns become eight operands without a transposition. K's lanes take the head's dims in an
// order of their own, which q's registers follow.
//
// The running maximum is a reference 2^11 under it, raised only where a weight would pass 2^15:
// weights stay within an f16, their low parts well above its smallest, and most tiles raise
// nothing.
//
// attn_q4_row: at most 16 query rows a KV head (a decode step, a short verify pass of few heads):
// a wave takes tiles of 32 slots of its workgroup's chunk, its four waves' states meet in LDS. Up
// to eight query rows put q's and the weights' two parts side by side in the MFMA's 16 columns:
// half the matrix work. attn_q4_tile: more query rows: a workgroup unpacks each tile of 64 slots
// once, into LDS in the order of the operands, and its waves take 16 or 32 query rows each.
// Chunks of a list meet in attn_q4_fold.
#include "common.hpp"
#include "internal.hpp"
#include "q4.hpp"

#include <hip/hip_ext.h>

#include <algorithm>
#include <type_traits>

namespace bchip {

// A sequence's rows over its cache: row r of the item (q and out row row0 + r) sees the slots
// below base + r (a line), or those below base and the named ones (a tree). Each of its lists is
// cut into nchunk chunks of `chunk` tiles.
struct Q4Item {
    uint32_t row0, rows, base, unit0, block0, nchunk, chunk, pad;
    uint64_t kvoff;
};

struct Q4Params {
    const float* q;
    const uint8_t* kc;
    const uint8_t* vc;
    float* out;
    float* part_o;   // [unit][QT][HD]: chunk states, QT query rows a unit
    float* part_ml;  // [unit][QT][2]: their references and sums
    const uint32_t* masks;
    uint32_t tree;
    uint32_t nh, nkv, G;
    uint32_t nqt;  // units of query rows a KV head (attn_q4_tile)
    uint32_t qt;   // query rows a unit (the fold)
    float sc;      // scale * log2(e)
    uint64_t slot_limit;
    uint32_t nitems;
    Q4Item items[MAX_ITEMS];
};

namespace {

constexpr float Q4_BIAS = 11.0f;  // log2 of the weight of a row's largest score when ref is set
constexpr float Q4_MOST = 15.0f;  // of any weight: an f16 holds it

// Two values of a word pair's 4-bit field k (bits 4k .. 4k + 3 of each half) times their scales.
__device__ __forceinline__ uint32_t unpack2(uint32_t w, int k, half2 d, half2 c) {
    const uint32_t f = k == 0 ? w << 4 : k == 1 ? w : k == 2 ? w >> 4 : w >> 8;
    const half2 x = __builtin_bit_cast(half2, (f & 0x00f000f0u) | 0x54005400u);  // 64 + code
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(x, d, c));
}

__device__ __forceinline__ half8 as_half8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_bit_cast(half8, uint4{a, b, c, d});
}

// A K operand's eight dims from their word: elements 0, 4, 1, 5, 2, 6, 3, 7.
__device__ __forceinline__ half8 unpack_k(uint32_t w, f16 scale) {
    const half2 d = {scale, scale}, c = d * (f16)-72.0f;
    return as_half8(unpack2(w, 0, d, c), unpack2(w, 1, d, c), unpack2(w, 2, d, c), unpack2(w, 3, d, c));
}

__device__ __forceinline__ bool odd_scale(f16 d) {  // an infinity or a NaN
    return (__builtin_bit_cast(uint16_t, d) & 0x7c00u) == 0x7c00u;
}

// V's columns of a head of 32 NB dims, in segments of 128, 64 and 32: a lane holds W consecutive
// columns of a segment.
template <int NB>
struct Seg {
    static constexpr int N128 = NB / 4, H64 = (NB % 4) >= 2, H32 = NB % 2, N = N128 + H64 + H32;
    static constexpr int w(int s) { return s < N128 ? 8 : (H64 && s == N128) ? 4 : 2; }
    static constexpr int col(int s) { return s < N128 ? 128 * s : (H64 && s == N128) ? 128 * N128 : 32 * (NB - 1); }
    static constexpr int frag(int s) { return s < N128 ? 8 * s : (H64 && s == N128) ? 8 * N128 : 8 * N128 + 4 * H64; }
};

template <int W>
__device__ __forceinline__ uint32_t load_codes(const uint8_t* p) {
    if constexpr (W == 8) return *(const uint32_t*)p;
    else if constexpr (W == 4) return *(const uint16_t*)p;
    else return *p;
}

// Operands of W columns from the words of eight slots and their scales.
template <int W>
__device__ __forceinline__ void unpack_v(const uint32_t (&raw)[8], const f16 (&sc)[8], half8 (&out)[W]) {
    uint32_t r[W][4];
#pragma unroll
    for (int p = 0; p < 4; p++) {
        const half2 d = {sc[2 * p], sc[2 * p + 1]}, c = d * (f16)-72.0f;
        const uint32_t lo = __builtin_amdgcn_perm(raw[2 * p + 1], raw[2 * p], 0x05040100u);
#pragma unroll
        for (int k = 0; k < (W < 4 ? W : 4); k++) r[k][p] = unpack2(lo, k, d, c);
        if constexpr (W == 8) {
            const uint32_t hi = __builtin_amdgcn_perm(raw[2 * p + 1], raw[2 * p], 0x07060302u);
#pragma unroll
            for (int k = 0; k < 4; k++) r[4 + k][p] = unpack2(hi, k, d, c);
        }
    }
#pragma unroll
    for (int k = 0; k < W; k++) out[k] = as_half8(r[k][0], r[k][1], r[k][2], r[k][3]);
}

// A lane's dims of one query row (8 words of NB, dims 8 (NB g + j) ..) as two f16 parts; back
// comes the power of two that scores are to be multiplied by.
template <int NB>
__device__ __forceinline__ float load_q(const float* qrow, uint32_t g, float sc, half8 (&hi)[NB], half8 (&lo)[NB]) {
    float x[NB][8];
    float top = 0.0f;
#pragma unroll
    for (int j = 0; j < NB; j++) {
        float4 a{}, b{};
        if (qrow) {
            a = *(const float4*)(qrow + 8 * (NB * g + j));
            b = *(const float4*)(qrow + 8 * (NB * g + j) + 4);
        }
        const float v[8] = {a.x, b.x, a.y, b.y, a.z, b.z, a.w, b.w};
#pragma unroll
        for (int i = 0; i < 8; i++) {
            x[j][i] = v[i] * sc;
            top = fmaxf(top, fabsf(x[j][i]));
        }
    }
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    int e = (int)(__float_as_uint(top) >> 23) - 127;  // (of an infinity 128: its row is NaN)
    e = e < -100 ? -100 : e;
    const float up = __uint_as_float((uint32_t)(13 - e + 127) << 23);
#pragma unroll
    for (int j = 0; j < NB; j++)
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float y = x[j][i] * up;
            hi[j][i] = (f16)y;
            lo[j][i] = (f16)(y - (float)hi[j][i]);
        }
    return __uint_as_float((uint32_t)(e - 13 + 127) << 23);
}

// Byte offsets, within a tile, of what a lane reads of a slot: its K words and scales.
template <int NB>
struct KLoad {
    static constexpr bool WHOLE = NB == 1 || NB == 2 || NB == 4 || NB == 8;  // consecutive bytes
    static constexpr int NC = WHOLE ? 1 : NB;                                // code offsets
    static constexpr int NS = NB == 8 ? 2 : WHOLE ? 1 : NB;                  // scales
    uint32_t code[NC], scale[NC];
    __device__ __forceinline__ void set(uint32_t e, uint32_t g) {
#pragma unroll
        for (int j = 0; j < NC; j++) {
            code[j] = q4_code_at32(e + 8 * (NB * g + j));
            scale[j] = q4_scale_at32(e + 8 * (NB * g + j));
        }
    }
    __device__ __forceinline__ void load(const uint8_t* tile, uint32_t (&w)[NB], f16 (&s)[NS]) const {
        if constexpr (NB == 1) {
            w[0] = *(const uint32_t*)(tile + code[0]);
        } else if constexpr (NB == 2) {
            const uint2 a = *(const uint2*)(tile + code[0]);
            w[0] = a.x, w[1] = a.y;
        } else if constexpr (NB == 4 || NB == 8) {
#pragma unroll
            for (int j = 0; j < NB; j += 4) {
                const uint4 a = *(const uint4*)(tile + code[0] + 4 * j);
                w[j] = a.x, w[j + 1] = a.y, w[j + 2] = a.z, w[j + 3] = a.w;
            }
        } else {
#pragma unroll
            for (int j = 0; j < NB; j++) w[j] = *(const uint32_t*)(tile + code[j]);
        }
        if constexpr (NB == 8) {
            const half2 a = *(const half2*)(tile + scale[0]);  // blocks 2g, 2g + 1
            s[0] = a[0], s[1] = a[1];
        } else {
#pragma unroll
            for (int j = 0; j < NS; j++) s[j] = *(const f16*)(tile + scale[j]);
        }
    }
    static __device__ __forceinline__ f16 of(const f16 (&s)[NS], int j) { return s[NB == 8 ? j / 4 : NS == 1 ? 0 : j]; }
};

// What query row n (of an item's rows x G) of this lane sees.
struct Sees {
    uint32_t vis;     // slots below this
    uint32_t lo, hi;  // a tree: and these from `base` on
    __device__ __forceinline__ bool at(uint32_t slot, uint32_t base, uint32_t end, uint32_t tree) const {
        if (slot >= end) return false;
        if (slot < vis) return true;
        if (!tree) return false;
        const uint32_t j = slot - base;
        return j < 64 && (((j < 32 ? lo >> j : hi >> (j - 32)) & 1u) != 0);
    }
};

// The end of an item's farthest list. A tree's is its highest named slot's: no slot past that is
// read. Every lane of the wave calls it.
__device__ __forceinline__ uint32_t tree_end(const Q4Params& p, const Q4Item& it) {
    const uint32_t lane = threadIdx.x & 63;
    uint32_t top = 0;
    if (lane < it.rows) {
        const uint32_t lo = p.masks[2 * (it.row0 + lane)], hi = p.masks[2 * (it.row0 + lane) + 1];
        top = hi ? 64 - __builtin_clz(hi) : lo ? 32 - __builtin_clz(lo) : 0;
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) top = max(top, (uint32_t)__shfl_xor((int)top, d));
    return (uint32_t)min((uint64_t)it.base + top, p.slot_limit);
}

// A row's weights are 2^(s - ref). Where some score of these 32 slots passes ref by more than
// Q4_MOST, the refs rise to Q4_BIAS under their rows' maxima (to the maxima themselves where
// those are so large that the difference would be lost), and what was summed against the old one
// is to be multiplied by f.
__device__ __forceinline__ bool raise(const float (&s)[8], float& ref, float& f) {
    float top = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7])));
    if (!__any(top > ref + Q4_MOST)) return false;
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    const float to = fmaxf(ref, fabsf(top) < 0x1p23f ? top - Q4_BIAS : top);
    f = to == -INFINITY ? 1.0f : exp2_hw(ref - to);
    ref = to;
    return true;
}

__device__ __forceinline__ float ror8(float x) {  // lane n of each 16 gets lane (n + 8) % 16's
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x128, 0xf, 0xf, false));
}

constexpr int Q4_WAVES = 4;
constexpr uint32_t Q4_TILE = 32;

template <int NB, bool PK>
__global__ __launch_bounds__(64 * Q4_WAVES) void attn_q4_row(const Q4Params p) {
    constexpr int HD = 32 * NB, NF = 2 * NB, ROWS = PK ? 8 : 16, LD = HD + 4;
    using S = Seg<NB>;
    __shared__ float so[Q4_WAVES][ROWS][LD];
    __shared__ float sm[Q4_WAVES][16], sl[Q4_WAVES][16];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m16 = lane & 15, g = lane >> 4;

    uint32_t ii = 0;
    if (p.nitems > 1) {  // the last item whose first block is at most this one
        const bool before = lane < p.nitems && p.items[lane].block0 <= blockIdx.x;
        ii = __builtin_amdgcn_readfirstlane(__popcll(__ballot(before)) - 1);
    }
    const Q4Item& it = p.items[ii];
    // Blocks 8 apart (one XCD) take the KV heads of one chunk: their bytes share cache lines.
    const uint32_t b = blockIdx.x - it.block0, oct = b / (8 * p.nkv), rest = b % (8 * p.nkv);
    const uint32_t kvh = rest / 8, chunk = oct * 8 + rest % 8;
    if (chunk >= it.nchunk) return;
    const uint32_t kvd = p.nkv * HD, nq = it.rows * p.G, end = p.tree ? tree_end(p, it) : it.base + it.rows - 1;

    const uint32_t n = PK ? (m16 & 7) : m16;
    const bool valid = n < nq;
    const uint32_t row = it.row0 + (valid ? n / p.G : 0), head = kvh * p.G + (valid ? n % p.G : 0);
    Sees see{valid ? it.base + (p.tree ? 0 : n / p.G) : end, 0, 0};
    if (p.tree && valid) {
        see.lo = p.masks[2 * row];
        see.hi = p.masks[2 * row + 1];
    }
    half8 qa[NB], qb[NB];
    const float c = load_q<NB>(valid ? p.q + ((size_t)row * p.nh + head) * HD : nullptr, g, p.sc, qa, qb);
    if constexpr (PK) {
#pragma unroll
        for (int j = 0; j < NB; j++)
            if (m16 >= 8) qa[j] = qb[j];
    }

    const uint64_t e0 = it.kvoff * kvd;
    const uint32_t rem = (uint32_t)(e0 & 255) + kvh * HD;
    const uint64_t tile_bytes = (uint64_t)kvd * 18;  // 32 slots
    const uint8_t* kbase = p.kc + (e0 >> 8) * Q4_UNIT_BYTES;
    const uint8_t* vbase = p.vc + (e0 >> 8) * Q4_UNIT_BYTES;

    const uint32_t ntiles = (uint32_t)(((uint64_t)end + Q4_TILE - 1) / Q4_TILE);
    const uint32_t t0 = chunk * it.chunk, t1 = min(t0 + it.chunk, ntiles);
    KLoad<NB> kl[2];
    uint32_t vcode[S::N][8], vscale[S::N][8];
    auto place = [&](uint32_t last) {  // slots past `last` read it instead (their weights are 0)
#pragma unroll
        for (int r = 0; r < 2; r++) kl[r].set(rem + min(16 * r + m16, last) * kvd, g);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint32_t e = rem + min(4 * g + (i & 3) + 16 * (i >> 2), last) * kvd;
#pragma unroll
            for (int si = 0; si < S::N; si++) {
                const uint32_t ec = e + S::col(si) + S::w(si) * m16;
                vcode[si][i] = q4_code_at32(ec);
                vscale[si][i] = q4_scale_at32(ec);
            }
        }
    };
    place(Q4_TILE - 1);

    f32x4 o[NF];
#pragma unroll
    for (int f = 0; f < NF; f++) o[f] = f32x4{0, 0, 0, 0};
    float ref = -INFINITY, l = 0.0f;

    for (uint32_t t = t0 + wave; t < t1; t += Q4_WAVES) {
        const uint32_t ts = t * Q4_TILE;
        if (end - ts < Q4_TILE) place(end - 1 - ts);
        const uint8_t* kt = kbase + t * tile_bytes;
        const uint8_t* vt = vbase + t * tile_bytes;
        uint32_t kw[2][NB], vw[S::N][8];
        f16 ks[2][KLoad<NB>::NS], vs[S::N][8];
#pragma unroll
        for (int r = 0; r < 2; r++) kl[r].load(kt, kw[r], ks[r]);
#pragma unroll
        for (int si = 0; si < S::N; si++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                vw[si][i] = S::w(si) == 8   ? load_codes<8>(vt + vcode[si][i])
                            : S::w(si) == 4 ? load_codes<4>(vt + vcode[si][i])
                                            : load_codes<2>(vt + vcode[si][i]);
                vs[si][i] = *(const f16*)(vt + vscale[si][i]);
            }
        float s[8];
#pragma unroll
        for (int r = 0; r < 2; r++) {
            f32x4 acc = {0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < NB; j++) {
                const half8 k = unpack_k(kw[r][j], KLoad<NB>::of(ks[r], j));
                acc = mfma16(k, qa[j], acc);
                if constexpr (!PK) acc = mfma16(k, qb[j], acc);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if constexpr (PK) acc[i] += ror8(acc[i]);
                s[4 * r + i] = acc[i] * c;
            }
        }
        // A tile that some row does not see whole: scores of unseen slots become -inf, and V
        // scales that are not finite 0, their blocks put back as NaN for the rows that see them.
        const bool edge = ts + Q4_TILE > it.base;
        bool odd = false;
        if (edge) {
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (!see.at(ts + 16 * (i >> 2) + 4 * g + (i & 3), it.base, end, p.tree)) s[i] = -INFINITY;
#pragma unroll
            for (int si = 0; si < S::N; si++)
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (odd_scale(vs[si][i])) {
                        vs[si][i] = (f16)0.0f;
                        odd = true;
                    }
        }
        float f;
        if (raise(s, ref, f)) {
            l *= f;
#pragma unroll
            for (int k = 0; k < NF; k++) o[k] *= f;
        }
        const float base = ref == -INFINITY ? 0.0f : ref;
        half8 ph, pl;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float w = exp2_hw(s[i] - base);
            l += w;
            const f16 h = (f16)w;
            if constexpr (PK) {
                ph[i] = m16 < 8 ? h : (f16)(w - (float)h);
            } else {
                ph[i] = h;
                pl[i] = (f16)(w - (float)h);
            }
        }
        auto pv = [&](auto width, int si) {
            constexpr int W = decltype(width)::value;
            half8 vf[W];
            unpack_v<W>(vw[si], vs[si], vf);
#pragma unroll
            for (int k = 0; k < W; k++) {
                f32x4& acc = o[S::frag(si) + k];
                acc = mfma16(vf[k], ph, acc);
                if constexpr (!PK) acc = mfma16(vf[k], pl, acc);
            }
        };
#pragma unroll
        for (int si = 0; si < S::N; si++) {
            if (S::w(si) == 8) pv(std::integral_constant<int, 8>{}, si);
            else if (S::w(si) == 4) pv(std::integral_constant<int, 4>{}, si);
            else pv(std::integral_constant<int, 2>{}, si);
        }
        if (edge && __any(odd)) {
            for (uint32_t i = 0; i < Q4_TILE && ts + i < end; i++) {
                const bool seen = see.at(ts + i, it.base, end, p.tree);
#pragma unroll
                for (int si = 0; si < S::N; si++) {  // (a lane's columns of a segment lie in one block)
                    const uint32_t e = rem + i * kvd + S::col(si) + S::w(si) * 4 * g;
                    if (seen && odd_scale(*(const f16*)(vt + q4_scale_at32(e))))
#pragma unroll
                        for (int k = 0; k < S::w(si); k++) o[S::frag(si) + k] = f32x4{NAN, NAN, NAN, NAN};
                }
            }
        }
    }

    // The four waves' states.
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if constexpr (PK) {
#pragma unroll
        for (int f = 0; f < NF; f++)
#pragma unroll
            for (int i = 0; i < 4; i++) o[f][i] += ror8(o[f][i]);
    }
    if (lane < 16) {
        sm[wave][lane] = ref;
        sl[wave][lane] = l;
    }
    if (valid && m16 < ROWS) {
#pragma unroll
        for (int si = 0; si < S::N; si++)
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int k = 0; k < S::w(si); k++)
                    so[wave][m16][S::col(si) + S::w(si) * (4 * g + i) + k] = o[S::frag(si) + k][i];
    }
    __syncthreads();
    const uint32_t unit = it.unit0 + kvh * it.nchunk + chunk;
    for (uint32_t x = threadIdx.x; x < nq * (HD / 4); x += 64 * Q4_WAVES) {
        const uint32_t r = x / (HD / 4), col = 4 * (x % (HD / 4));
        float M = sm[0][r];
#pragma unroll
        for (int w = 1; w < Q4_WAVES; w++) M = fmaxf(M, sm[w][r]);
        const float Ms = M == -INFINITY ? 0.0f : M;
        float L = 0.0f;
        f32x4 a = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < Q4_WAVES; w++) {
            const float k = exp2_hw(sm[w][r] - Ms);
            L += k * sl[w][r];
            a += k * *(const f32x4*)&so[w][r][col];
        }
        if (it.nchunk == 1) {
            const float inv = L == 0.0f ? 0.0f : 1.0f / L;  // (a row that sees nothing: zeros)
            const uint32_t orow = it.row0 + r / p.G, oh = kvh * p.G + r % p.G;
            *(f32x4*)(p.out + ((size_t)orow * p.nh + oh) * HD + col) = a * inv;
        } else {
            *(f32x4*)(p.part_o + ((size_t)unit * 16 + r) * HD + col) = a;
            if (col == 0) {
                p.part_ml[2 * ((size_t)unit * 16 + r)] = M;
                p.part_ml[2 * ((size_t)unit * 16 + r) + 1] = L;
            }
        }
    }
}

// More query rows: a tile of 64 slots unpacked once into LDS for the workgroup's four waves of
// 16 RT query rows each.
constexpr uint32_t Q4_TILE_B = 64;

template <int NB, int RT>
__global__ __launch_bounds__(64 * Q4_WAVES, NB <= 4 ? 2 : 1) void attn_q4_tile(const Q4Params p) {
    constexpr int HD = 32 * NB, NF = 2 * NB;
    constexpr uint32_t QT = 64 * RT;
    using S = Seg<NB>;
    __shared__ half8 kf[2][4][NB][64];
    __shared__ half8 vf[2][2][NF][64];
    __shared__ uint32_t odd_tile[2];  // 1 + the tile of each buffer that held a scale that is not finite
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m16 = lane & 15, g = lane >> 4;
    const Q4Item& it = p.items[0];
    // Blocks 8 apart take one KV head's units of query rows, the longest lists first.
    uint32_t b = blockIdx.x;
    const uint32_t kvh = b % p.nkv;
    b /= p.nkv;
    const uint32_t qt = p.nqt - 1 - b / it.nchunk, chunk = b % it.nchunk;
    const uint32_t kvd = p.nkv * HD, nq = it.rows * p.G, q0 = qt * QT, q1 = min(q0 + QT, nq);
    const uint32_t first = p.tree ? it.base : it.base + q0 / p.G;  // slots every row here sees
    const uint32_t end = p.tree ? tree_end(p, it) : it.base + (q1 - 1) / p.G;

    Sees see[RT];
    half8 qh[RT][NB], ql[RT][NB];
    float c[RT];
#pragma unroll
    for (int r = 0; r < RT; r++) {
        const uint32_t n = q0 + (wave * RT + r) * 16 + m16;
        const bool valid = n < nq;
        const uint32_t row = it.row0 + (valid ? n / p.G : 0), head = kvh * p.G + (valid ? n % p.G : 0);
        see[r] = Sees{valid ? it.base + (p.tree ? 0 : n / p.G) : end, 0, 0};
        if (p.tree && valid) {
            see[r].lo = p.masks[2 * row];
            see[r].hi = p.masks[2 * row + 1];
        }
        c[r] = load_q<NB>(valid ? p.q + ((size_t)row * p.nh + head) * HD : nullptr, g, p.sc, qh[r], ql[r]);
    }

    const uint64_t e0 = it.kvoff * kvd;
    const uint32_t rem = (uint32_t)(e0 & 255) + kvh * HD;
    const uint64_t tile_bytes = (uint64_t)kvd * 36;  // 64 slots
    const uint8_t* kbase = p.kc + (e0 >> 8) * Q4_UNIT_BYTES;
    const uint8_t* vbase = p.vc + (e0 >> 8) * Q4_UNIT_BYTES;
    const uint32_t ntiles = (uint32_t)(((uint64_t)end + Q4_TILE_B - 1) / Q4_TILE_B);
    const uint32_t t0 = chunk * it.chunk, t1 = min(t0 + it.chunk, ntiles);

    // This wave's share of a tile: K's slots 16 wave .. + 15, and of V's half wave / 2 half the
    // columns of every lane.
    const uint32_t half = wave & 1, step = wave >> 1;
    KLoad<NB> kl;
    uint32_t vcode[S::N][8], vscale[S::N][8];
    auto place = [&](uint32_t last) {
        kl.set(rem + min(16 * wave + m16, last) * kvd, g);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint32_t e = rem + min(32 * step + 4 * g + (i & 3) + 16 * (i >> 2), last) * kvd;
#pragma unroll
            for (int si = 0; si < S::N; si++) {
                const uint32_t W = S::w(si), ec = e + S::col(si) + W * m16 + (W == 2 ? 0 : W / 2 * half);
                vcode[si][i] = q4_code_at32(ec);
                vscale[si][i] = q4_scale_at32(ec);
            }
        }
    };
    place(Q4_TILE_B - 1);
    uint32_t kw[NB], vw[S::N][8];
    f16 ks[KLoad<NB>::NS], vs[S::N][8];
    auto fetch = [&](uint32_t t) {
        const uint32_t ts = t * Q4_TILE_B;
        if (end - ts < Q4_TILE_B) place(end - 1 - ts);
        const uint8_t* kt = kbase + t * tile_bytes;
        const uint8_t* vt = vbase + t * tile_bytes;
        kl.load(kt, kw, ks);
#pragma unroll
        for (int si = 0; si < S::N; si++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                vw[si][i] = S::w(si) == 8 ? load_codes<4>(vt + vcode[si][i]) : load_codes<2>(vt + vcode[si][i]);
                vs[si][i] = *(const f16*)(vt + vscale[si][i]);
            }
    };
    auto unpack = [&](uint32_t t, int buf) {
        if (t * Q4_TILE_B + Q4_TILE_B > first) {  // some row here does not see all of it
            bool odd = false;
#pragma unroll
            for (int si = 0; si < S::N; si++)
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (odd_scale(vs[si][i])) {
                        vs[si][i] = (f16)0.0f;
                        odd = true;
                    }
            if (odd) odd_tile[buf] = t + 1;
        }
#pragma unroll
        for (int j = 0; j < NB; j++) kf[buf][wave][j][lane] = unpack_k(kw[j], KLoad<NB>::of(ks, j));
#pragma unroll
        for (int si = 0; si < S::N; si++) {
            if (S::w(si) == 8) {
                half8 x[4];
                unpack_v<4>(vw[si], vs[si], x);
#pragma unroll
                for (int k = 0; k < 4; k++) vf[buf][step][S::frag(si) + 4 * half + k][lane] = x[k];
            } else if (S::w(si) == 4) {
                half8 x[2];
                unpack_v<2>(vw[si], vs[si], x);
#pragma unroll
                for (int k = 0; k < 2; k++) vf[buf][step][S::frag(si) + 2 * half + k][lane] = x[k];
            } else {
                half8 x[2];
                unpack_v<2>(vw[si], vs[si], x);
                vf[buf][step][S::frag(si) + half][lane] = half ? x[1] : x[0];
            }
        }
    };

    f32x4 o[RT][NF];
    float ref[RT], l[RT];
#pragma unroll
    for (int r = 0; r < RT; r++) {
        ref[r] = -INFINITY;
        l[r] = 0.0f;
#pragma unroll
        for (int f = 0; f < NF; f++) o[r][f] = f32x4{0, 0, 0, 0};
    }
    if (threadIdx.x < 2) odd_tile[threadIdx.x] = 0;
    if (t0 < t1) fetch(t0);
    __syncthreads();
    if (t0 < t1) unpack(t0, 0);
    __syncthreads();
    for (uint32_t t = t0; t < t1; t++) {
        const int buf = (t - t0) & 1;
        const uint32_t ts = t * Q4_TILE_B;
        if (t + 1 < t1) fetch(t + 1);
        const bool edge = ts + Q4_TILE_B > first;
#pragma unroll
        for (int u = 0; u < 2; u++) {
            f32x4 acc[RT][2];
#pragma unroll
            for (int r = 0; r < RT; r++) acc[r][0] = acc[r][1] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < NB; j++)
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    const half8 k = kf[buf][2 * u + x][j][lane];
#pragma unroll
                    for (int r = 0; r < RT; r++) {
                        acc[r][x] = mfma16(k, qh[r][j], acc[r][x]);
                        acc[r][x] = mfma16(k, ql[r][j], acc[r][x]);
                    }
                }
            half8 ph[RT], pl[RT];
#pragma unroll
            for (int r = 0; r < RT; r++) {
                float s[8];
#pragma unroll
                for (int i = 0; i < 8; i++) s[i] = acc[r][i >> 2][i & 3] * c[r];
                if (edge)
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        if (!see[r].at(ts + 32 * u + 16 * (i >> 2) + 4 * g + (i & 3), it.base, end, p.tree)) s[i] = -INFINITY;
                float f;
                if (raise(s, ref[r], f)) {
                    l[r] *= f;
#pragma unroll
                    for (int k = 0; k < NF; k++) o[r][k] *= f;
                }
                const float base = ref[r] == -INFINITY ? 0.0f : ref[r];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float w = exp2_hw(s[i] - base);
                    l[r] += w;
                    ph[r][i] = (f16)w;
                    pl[r][i] = (f16)(w - (float)ph[r][i]);
                }
            }
#pragma unroll
            for (int f = 0; f < NF; f++) {
                const half8 v = vf[buf][u][f][lane];
#pragma unroll
                for (int r = 0; r < RT; r++) {
                    o[r][f] = mfma16(v, ph[r], o[r][f]);
                    o[r][f] = mfma16(v, pl[r], o[r][f]);
                }
            }
        }
        if (edge && odd_tile[buf] == t + 1) {
            const uint8_t* vt = vbase + t * tile_bytes;
            for (uint32_t i = 0; i < Q4_TILE_B && ts + i < end; i++)
#pragma unroll
                for (int si = 0; si < S::N; si++) {
                    const uint32_t e = rem + i * kvd + S::col(si) + S::w(si) * 4 * g;
                    const bool odd = odd_scale(*(const f16*)(vt + q4_scale_at32(e)));
#pragma unroll
                    for (int r = 0; r < RT; r++)
                        if (odd && see[r].at(ts + i, it.base, end, p.tree))
#pragma unroll
                            for (int k = 0; k < S::w(si); k++) o[r][S::frag(si) + k] = f32x4{NAN, NAN, NAN, NAN};
                }
        }
        if (t + 1 < t1) unpack(t + 1, buf ^ 1);
        __syncthreads();
    }

    const uint32_t unit = (kvh * p.nqt + qt) * it.nchunk + chunk;
#pragma unroll
    for (int r = 0; r < RT; r++) {
        l[r] += __shfl_xor(l[r], 16);
        l[r] += __shfl_xor(l[r], 32);
        const uint32_t sl = (wave * RT + r) * 16 + m16, n = q0 + sl;
        if (n >= nq) continue;
        float* dst;
        float k = 1.0f;
        if (it.nchunk == 1) {
            dst = p.out + ((size_t)(it.row0 + n / p.G) * p.nh + kvh * p.G + n % p.G) * HD;
            k = l[r] == 0.0f ? 0.0f : 1.0f / l[r];
        } else {
            dst = p.part_o + ((size_t)unit * QT + sl) * HD;
            if (g == 0) {
                p.part_ml[2 * ((size_t)unit * QT + sl)] = ref[r];
                p.part_ml[2 * ((size_t)unit * QT + sl) + 1] = l[r];
            }
        }
#pragma unroll
        for (int si = 0; si < S::N; si++)
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int x = 0; x < S::w(si); x++)
                    dst[S::col(si) + S::w(si) * (4 * g + i) + x] = o[r][S::frag(si) + x][i] * k;
    }
}

// One output row of one head from its chunks' states.
constexpr uint32_t Q4_MAX_CHUNKS = 256;

__global__ __launch_bounds__(256) void attn_q4_fold(const Q4Params p, uint32_t hd) {
    __shared__ float wt[Q4_MAX_CHUNKS];
    __shared__ float red[8];
    __shared__ f32x4 sum[256];
    const uint32_t tid = threadIdx.x, head = blockIdx.x, kvh = head / p.G;
    const Q4Item& it = p.items[p.nitems > 1 ? blockIdx.y : 0];
    if (it.nchunk == 1) return;  // written by its workgroup
    const uint32_t r = p.nitems > 1 ? 0 : blockIdx.y, n = r * p.G + head % p.G;
    const size_t u0 = it.unit0 + (size_t)(kvh * p.nqt + n / p.qt) * it.nchunk;
    const uint32_t sl = n % p.qt;
    float mc = -INFINITY, lc = 0.0f;
    if (tid < it.nchunk) {
        const float2 ml = *(const float2*)(p.part_ml + 2 * ((u0 + tid) * p.qt + sl));
        mc = ml.x;
        lc = ml.y;
    }
    float M = mc;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) M = fmaxf(M, __shfl_xor(M, d));
    if ((tid & 63) == 0) red[tid >> 6] = M;
    __syncthreads();
    M = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float w = exp2_hw(mc - (M == -INFINITY ? 0.0f : M));
    wt[tid] = w;
    float L = w * lc;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) L += __shfl_xor(L, d);
    if ((tid & 63) == 0) red[4 + (tid >> 6)] = L;
    __syncthreads();
    L = (red[4] + red[5]) + (red[6] + red[7]);
    const uint32_t q = hd / 4, parts = 256 / q, part = tid / q, col = 4 * (tid % q);
    f32x4 a = {0, 0, 0, 0};
    if (part < parts)
        for (uint32_t c = part; c < it.nchunk; c += parts)
            a += wt[c] * *(const f32x4*)(p.part_o + ((u0 + c) * p.qt + sl) * hd + col);
    sum[tid] = a;
    __syncthreads();
    if (part == 0) {
        for (uint32_t k = 1; k < parts; k++) a += sum[k * q + tid];
        *(f32x4*)(p.out + ((size_t)(it.row0 + r) * p.nh + head) * hd + col) = a * (L == 0.0f ? 0.0f : 1.0f / L);
    }
}

template <int NB>
void launch_row(const Q4Params& p, uint32_t blocks, bool pk, const AttnCall& a, hipStream_t s) {
    const dim3 grid(blocks), wg(64 * Q4_WAVES);
    if (pk) hipExtLaunchKernelGGL((attn_q4_row<NB, true>), grid, wg, 0, s, a.ev_before, a.ev_after, 0, p);
    else hipExtLaunchKernelGGL((attn_q4_row<NB, false>), grid, wg, 0, s, a.ev_before, a.ev_after, 0, p);
}
template <int NB>
void launch_tile(const Q4Params& p, uint32_t blocks, uint32_t rt, const AttnCall& a, hipStream_t s) {
    const dim3 grid(blocks), wg(64 * Q4_WAVES);
    if constexpr (NB <= 4) {
        if (rt == 2) {
            hipExtLaunchKernelGGL((attn_q4_tile<NB, 2>), grid, wg, 0, s, a.ev_before, a.ev_after, 0, p);
            return;
        }
    }
    hipExtLaunchKernelGGL((attn_q4_tile<NB, 1>), grid, wg, 0, s, a.ev_before, a.ev_after, 0, p);
}

Q4Params params(const AttnCall& a) {
    Q4Params p{};
    p.q = a.q;
    p.kc = (const uint8_t*)a.kc;
    p.vc = (const uint8_t*)a.vc;
    p.out = a.out;
    p.masks = a.masks;
    p.tree = a.tree;
    p.nh = a.nh;
    p.nkv = a.nkv;
    p.G = a.nh / a.nkv;
    p.sc = a.scale * LOG2E;
    p.slot_limit = a.slot_limit;
    p.nqt = 1;
    p.qt = 16;
    return p;
}

// Workgroups of attn_q4_row that keep the GPU busy: chunks of a list are made to come near it.
constexpr uint32_t Q4_ROW_GROUPS = 1024;
constexpr uint32_t Q4_TILE_GROUPS = 512;

// Chunks for a list of `tiles` tiles, `least` at least a chunk, for `want` of them.
void cut(Q4Item& it, uint64_t tiles, uint32_t want, uint32_t least) {
    const uint64_t n = std::max<uint64_t>(1, std::min<uint64_t>({(uint64_t)want, tiles / least, Q4_MAX_CHUNKS}));
    it.chunk = (uint32_t)std::max<uint64_t>(1, (tiles + n - 1) / n);
    it.nchunk = (uint32_t)std::max<uint64_t>(1, (tiles + it.chunk - 1) / it.chunk);
}

bool reserve(Q4Params& p, uint64_t states, uint32_t hd, Workspace& ws, hipStream_t s) {
    const bool had = ws.reserve_if(states, hd <= 32 ? 32 : hd <= 64 ? 64 : hd <= 128 ? 128 : 256, s);
    p.part_o = ws.o;
    p.part_ml = ws.ml;
    return had;
}

#define Q4_BY_DIM(nb, call)     \
    switch (nb) {               \
        case 1: call(1); break; \
        case 2: call(2); break; \
        case 3: call(3); break; \
        case 4: call(4); break; \
        case 5: call(5); break; \
        case 6: call(6); break; \
        case 7: call(7); break; \
        default: call(8);       \
    }

// One launch of attn_q4_row over p's items of `lens` entries, and the fold of its chunks. A
// call whose scratch cannot be had takes each list in one chunk.
hipError_t launch_items(Q4Params& p, const AttnCall& a, const uint64_t* lens, Workspace& ws, hipStream_t s) {
    uint64_t total = 0;
    for (uint32_t i = 0; i < p.nitems; i++) total += (lens[i] + Q4_TILE - 1) / Q4_TILE;
    const uint32_t want = std::max(1u, Q4_ROW_GROUPS / a.nkv);
    uint32_t units, blocks;
    bool split;
    auto plan = [&](uint64_t all) {
        units = blocks = 0;
        split = false;
        for (uint32_t i = 0; i < p.nitems; i++) {
            Q4Item& it = p.items[i];
            const uint64_t tiles = (lens[i] + Q4_TILE - 1) / Q4_TILE;
            it.unit0 = units;
            it.block0 = blocks;
            // A list's share of the workgroups is its share of the tiles.
            cut(it, tiles, (uint32_t)std::max<uint64_t>(1, all * tiles / std::max<uint64_t>(1, total)), Q4_WAVES);
            units += it.nchunk * a.nkv;
            blocks += (it.nchunk + 7) / 8 * 8 * a.nkv;
            split |= it.nchunk > 1;
        }
    };
    plan(want);
    if (split && !reserve(p, (uint64_t)units * 16, a.hd, ws, s)) plan(0);
    const bool pk = p.items[0].rows * p.G <= 8;
#define Q4_ROW(NB) launch_row<NB>(p, blocks, pk, a, s)
    Q4_BY_DIM(a.hd / 32, Q4_ROW)
#undef Q4_ROW
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || !split) return e;
    hipLaunchKernelGGL(attn_q4_fold, dim3(a.nh, p.nitems > 1 ? p.nitems : a.rows), dim3(256), 0, s, p, a.hd);
    return hipGetLastError();
}

}  // namespace

hipError_t q4_attention(const AttnCall& a, Workspace& ws, hipStream_t s) {
    Q4Params p = params(a);
    Q4Item& it = p.items[0];
    p.nitems = 1;
    it.rows = a.rows;
    it.base = a.tree ? a.pos : a.pos + 1;
    const uint64_t far = std::min<uint64_t>((uint64_t)a.pos + (a.tree ? 64 : a.rows), a.slot_limit);
    const uint64_t nq = (uint64_t)a.rows * p.G;
    if (nq <= 16) return launch_items(p, a, &far, ws, s);
    // 32 query rows a wave where that still makes a workgroup for every CU.
    const uint32_t rt = a.hd <= 128 && (nq + 127) / 128 * a.nkv >= 256 ? 2 : 1;
    p.qt = 64 * rt;
    p.nqt = (uint32_t)((nq + p.qt - 1) / p.qt);
    const uint64_t groups = (uint64_t)p.nqt * a.nkv, tiles = (far + Q4_TILE_B - 1) / Q4_TILE_B;
    cut(it, tiles, (uint32_t)std::max<uint64_t>(1, Q4_TILE_GROUPS / groups), 2);
    if (it.nchunk > 1 && !reserve(p, groups * it.nchunk * p.qt, a.hd, ws, s)) cut(it, tiles, 1, 2);
    const uint64_t blocks = groups * it.nchunk;
    if (blocks > 0x7fffffffull) return hipErrorInvalidValue;
#define Q4_TILES(NB) launch_tile<NB>(p, (uint32_t)blocks, rt, a, s)
    Q4_BY_DIM(a.hd / 32, Q4_TILES)
#undef Q4_TILES
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || it.nchunk == 1) return e;
    hipLaunchKernelGGL(attn_q4_fold, dim3(a.nh, a.rows), dim3(256), 0, s, p, a.hd);
    return hipGetLastError();
}

hipError_t q4_attention_ragged(const AttnCall& a, const uint32_t* lens, const uint64_t* offs, uint32_t nseq,
                               Workspace& ws, hipStream_t s) {
    AttnCall call = a;
    call.rows = 1;
    for (uint32_t s0 = 0; s0 < nseq; s0 += MAX_ITEMS) {
        Q4Params p = params(a);
        p.nitems = std::min<uint32_t>(MAX_ITEMS, nseq - s0);
        uint64_t len[MAX_ITEMS];
        for (uint32_t i = 0; i < p.nitems; i++) {
            Q4Item& it = p.items[i];
            it.row0 = s0 + i;
            it.rows = 1;
            it.base = lens[s0 + i];
            it.kvoff = offs[s0 + i];
            len[i] = lens[s0 + i];
        }
        const hipError_t e = launch_items(p, call, len, ws, s);
        if (e != hipSuccess) return e;
        call.ev_before = call.ev_after = nullptr;
    }
    return hipSuccess;
}

}  // namespace bchip
