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
// a wave takes tiles of 32 slots of its workgroup's chunk, the waves' states meet in LDS. Up
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
// cut into nchunk chunks of `chunk` tiles; block0 is the first of its rows of eight blocks,
// turned by `turn` so that an item's first chunk lies behind the last of the item before.
struct Q4Item {
    uint32_t row0, rows, base, unit0, block0, nchunk, chunk, turn;
    uint64_t kvoff;
};

struct Q4Params {
    const float* q;
    const uint8_t* kc;
    const uint8_t* vc;
    float* out;
    float* part_o;   // [unit][qt / 16][HD / 16][64][4]: chunk states, qt query rows a unit
    float* part_ml;  // [unit][qt][2]: their references and sums
    const uint32_t* masks;
    uint32_t tree;
    uint32_t nh, nkv, G;
    uint32_t nqt;  // units of query rows a KV head (attn_q4_tile)
    uint32_t qt;   // query rows a unit
    float sc;      // scale * log2(e)
    uint64_t slot_limit;
    uint32_t nitems;
    Q4Item items[MAX_ITEMS];
};

namespace {

constexpr float Q4_BIAS = 11.0f;  // log2 of the weight of a row's largest score when ref is set
constexpr float Q4_MOST = 15.0f;  // of any weight: an f16 holds it

// The constants of the unpacking, in registers so that one instruction takes both.
struct Q4Bits {
    uint32_t field, sixty4;
    __device__ __forceinline__ Q4Bits() {
        asm("v_mov_b32 %0, 0x00f000f0" : "=v"(field));
        asm("s_mov_b32 %0, 0x54005400" : "=s"(sixty4));
    }
};

// Two values of a word pair's 4-bit field k (bits 4k .. 4k + 3 of each half) times their scales.
__device__ __forceinline__ uint32_t unpack2(const Q4Bits& b, uint32_t w, int k, half2 d, half2 c) {
    const uint32_t f = k == 0 ? w << 4 : k == 1 ? w : k == 2 ? w >> 4 : w >> 8;
    const half2 x = __builtin_bit_cast(half2, (f & b.field) | b.sixty4);  // 64 + code
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(x, d, c));
}

__device__ __forceinline__ half8 as_half8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_bit_cast(half8, uint4{a, b, c, d});
}

// A K operand's eight dims from their word: elements 0, 4, 1, 5, 2, 6, 3, 7.
__device__ __forceinline__ half8 unpack_k(const Q4Bits& b, uint32_t w, f16 scale) {
    const half2 d = {scale, scale}, c = d * (f16)-72.0f;
    return as_half8(unpack2(b, w, 0, d, c), unpack2(b, w, 1, d, c), unpack2(b, w, 2, d, c), unpack2(b, w, 3, d, c));
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

// The columns of operand f that result registers 0 .. 3 of lane group g hold: the first, and how
// far they are apart.
template <int NB>
__device__ __forceinline__ uint32_t stride(uint32_t f) {
    using S = Seg<NB>;
    return f < 8u * S::N128 ? 8 : S::H64 && f < 8u * S::N128 + 4u ? 4 : 2;
}
template <int NB>
__device__ __forceinline__ uint32_t column(uint32_t f, uint32_t g) {
    using S = Seg<NB>;
    if (f < 8u * S::N128) return 128 * (f / 8) + f % 8 + 32 * g;
    if (S::H64 && f < 8u * S::N128 + 4u) return 128 * S::N128 + f % 4 + 16 * g;
    return 32 * (NB - 1) + f % 2 + 8 * g;
}

// Operands of W columns from the words of eight slots and their scales.
template <int W>
__device__ __forceinline__ void unpack_v(const Q4Bits& b, const uint32_t (&raw)[8], const f16 (&sc)[8], half8 (&out)[W]) {
    uint32_t r[W][4];
#pragma unroll
    for (int p = 0; p < 4; p++) {
        const half2 d = {sc[2 * p], sc[2 * p + 1]}, c = d * (f16)-72.0f;
        const uint32_t lo = __builtin_amdgcn_perm(raw[2 * p + 1], raw[2 * p], 0x05040100u);
#pragma unroll
        for (int k = 0; k < (W < 4 ? W : 4); k++) r[k][p] = unpack2(b, lo, k, d, c);
        if constexpr (W == 8) {
            const uint32_t hi = __builtin_amdgcn_perm(raw[2 * p + 1], raw[2 * p], 0x07060302u);
#pragma unroll
            for (int k = 0; k < 4; k++) r[4 + k][p] = unpack2(b, hi, k, d, c);
        }
    }
#pragma unroll
    for (int k = 0; k < W; k++) out[k] = as_half8(r[k][0], r[k][1], r[k][2], r[k][3]);
}

// The larger of two, a number before a NaN: fmaxf without the quieting of its operands.
__device__ __forceinline__ float larger(float a, float b) { return __builtin_amdgcn_fmed3f(a, b, INFINITY); }

typedef float f32x2 __attribute__((ext_vector_type(2)));

// Eight dims of a query row from `at`, in the order of a K word's.
__device__ __forceinline__ void q_load(const float* at, bool valid, float (&x)[8]) {
    float4 a{}, b{};
    if (valid) {
        a = *(const float4*)at;
        b = *(const float4*)(at + 4);
    }
    x[0] = a.x, x[1] = b.x, x[2] = a.y, x[3] = b.y, x[4] = a.z, x[5] = b.z, x[6] = a.w, x[7] = b.w;
}
// The largest magnitude of them and `top`.
__device__ __forceinline__ float q_top(const float (&x)[8], float top) {
#pragma unroll
    for (int i = 0; i < 8; i++) top = larger(top, fabsf(x[i]));
    return top;
}

// From a row's largest |q|: q times k is q scale log2 e brought to 2^13 .. 2^14, c takes it back.
__device__ __forceinline__ void q_scale(float top, float sc, float& k, float& c) {
    int e = (int)(__float_as_uint(top * fabsf(sc)) >> 23) - 127;  // (of an infinity 128: its row is NaN)
    e = e < -100 ? -100 : e;
    k = sc * __uint_as_float((uint32_t)(13 - e + 127) << 23);
    c = __uint_as_float((uint32_t)(e - 13 + 127) << 23);
}

__device__ __forceinline__ void q_parts(const float (&x)[8], float k, half8& hi, half8& lo) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const half2 h = __builtin_convertvector((f32x2{x[i] * k, x[i + 1] * k}), half2);
        const half2 r = __builtin_convertvector((f32x2{__builtin_fmaf(x[i], k, -(float)h[0]), __builtin_fmaf(x[i + 1], k, -(float)h[1])}), half2);
        hi[i] = h[0], hi[i + 1] = h[1];
        lo[i] = r[0], lo[i + 1] = r[1];
    }
}

// A list's codes and scales are read through buffer descriptors that end with its last slot's
// unit: what a tile reaches past that comes back as zero, whatever lies there.
typedef __amdgpu_buffer_rsrc_t q4_rsrc;
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ q4_rsrc q4_from(const uint8_t* base, uint64_t at, uint64_t end) {
    return __builtin_amdgcn_make_buffer_rsrc((void*)(base + at), 0, (uint32_t)min(end - at, (uint64_t)0x7fffffffu), 0x00020000);
}
__device__ __forceinline__ f16 load_scale(q4_rsrc r, uint32_t at) {
    return __builtin_bit_cast(f16, (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(r, at, 0, 0));
}

// One head's part of SLOTS slots of K or V on its way into LDS: a thread takes blocks of a slot,
// 16 bytes of codes and their scale, so consecutive lanes read consecutive bytes (loads of a few
// bytes a lane at the operands' own places cost the memory path 30 to 60 cycles each). In LDS a slot
// takes SLOT bytes, its codes and then its scales. For heads of 64, 128, 192 and 256 that is an odd
// multiple of 16, so the operands' lanes read every bank once. For heads of an odd number of blocks it is
// 32, 64, 96 or 128, and a group's lanes share banks (four of them start the 16 slots of heads of 96, two
// those of 224), a word at a time: 16 x 4 heads of 96, 160 and 224 take 9.1, 11.0 and 18.2 us for a step at
// 512 slots, the next even ones 8.0, 11.2 and 11.9; 2000 rows 60, 79 and 123, the next ones 60, 83 and 98.
// (Heads of 224 also spill: a vector register in a step's short form.)
template <int NB, int SLOTS, int THREADS>
struct Raw {
    static constexpr int SLOT = 16 * NB + 16, BYTES = SLOT * SLOTS;
    static constexpr int N = (SLOTS * NB + THREADS - 1) / THREADS, STEP = THREADS / NB;  // slots from load to load
    static constexpr bool SAME = THREADS % NB == 0 && STEP % 8 == 0;  // (8 slots are whole units)
    static constexpr int M = SAME ? 1 : N;
    uint32_t code[M], scale[M], to[M], tod[M];
    u32x4 c[N];
    uint16_t d[N];
    __device__ __forceinline__ void set(uint32_t rem, uint32_t kvd, uint32_t thread) {
#pragma unroll
        for (int i = 0; i < M; i++) {
            const uint32_t x = min((uint32_t)(i * THREADS) + thread, (uint32_t)(SLOTS * NB - 1)), slot = x / NB, b = x % NB;
            const uint32_t e = rem + slot * kvd + 32 * b;
            code[i] = q4_code_at32(e);
            scale[i] = q4_scale_at32(e);
            to[i] = slot * SLOT + 16 * b;
            tod[i] = slot * SLOT + 16 * NB + 2 * b;
        }
    }
    __device__ __forceinline__ void load(q4_rsrc r, uint32_t kvd) {
#pragma unroll
        for (int i = 0; i < N; i++) {
            const uint32_t at = SAME ? i * (STEP / 8) * (kvd / 2 * 9) : 0;
            c[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, code[SAME ? 0 : i], at, 0));
            d[i] = __builtin_amdgcn_raw_buffer_load_b16(r, scale[SAME ? 0 : i], at, 0);
        }
    }
    __device__ __forceinline__ void store(uint8_t* lds) const {
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int at = SAME ? i * STEP * SLOT : 0;
            *(u32x4*)(lds + to[SAME ? 0 : i] + at) = c[i];
            *(uint16_t*)(lds + tod[SAME ? 0 : i] + at) = d[i];
        }
    }
};

// K's operands of a slot in LDS: lane group g takes the words NB g .. NB g + NB - 1 of its codes.
template <int NB>
__device__ __forceinline__ void read_k(const uint8_t* slot, uint32_t g, uint32_t (&w)[NB], f16 (&s)[NB]) {
    constexpr int ALIGN = NB % 4 == 0 ? 4 : NB % 2 == 0 ? 2 : 1;
    if constexpr (ALIGN == 4) {
#pragma unroll
        for (int j = 0; j < NB; j += 4) {
            const u32x4 a = *(const u32x4*)(slot + 4 * (NB * g + j));
            w[j] = a.x, w[j + 1] = a.y, w[j + 2] = a.z, w[j + 3] = a.w;
        }
    } else if constexpr (ALIGN == 2) {
#pragma unroll
        for (int j = 0; j < NB; j += 2) {
            const u32x2 a = *(const u32x2*)(slot + 4 * (NB * g + j));
            w[j] = a.x, w[j + 1] = a.y;
        }
    } else {
#pragma unroll
        for (int j = 0; j < NB; j++) w[j] = *(const uint32_t*)(slot + 4 * (NB * g + j));
    }
    constexpr int SAME = NB == 1 || NB == 2 || NB == 4 || NB == 8 ? (NB < 4 ? NB : 4) : 1;  // words of one block
#pragma unroll
    for (int j = 0; j < NB; j++) s[j] = j % SAME ? s[j - 1] : *(const f16*)(slot + 16 * NB + 2 * ((NB * g + j) >> 2));
}

// W columns of V's segment si in LDS (W: the segment's, or half of them from the half'th on), for
// the operands of 32 slots from `tile`: slots 4g .. 4g + 3 and 16 + 4g ... .
template <int NB, bool HALF>
struct VRead {
    using S = Seg<NB>;
    static constexpr int w(int si) { return HALF && S::w(si) > 2 ? S::w(si) / 2 : S::w(si); }
    uint32_t word[S::N][8];
    f16 scale[S::N][8];
    __device__ __forceinline__ void read(const uint8_t* tile, uint32_t m16, uint32_t g, uint32_t half) {
        constexpr int SLOT = 16 * NB + 16;
#pragma unroll
        for (int si = 0; si < S::N; si++) {
            const uint32_t c = S::col(si) + S::w(si) * m16;
            const uint8_t* at = tile + 4 * g * SLOT;
            const uint32_t code = c / 2 + (w(si) < S::w(si) ? w(si) / 2 * half : 0), d = 16 * NB + c / 32 * 2;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const uint8_t* x = at + ((i & 3) + 16 * (i >> 2)) * SLOT;
                word[si][i] = w(si) == 8   ? *(const uint32_t*)(x + code)
                              : w(si) == 4 ? *(const uint16_t*)(x + code)
                                           : (uint32_t) * (x + code);
                scale[si][i] = *(const f16*)(x + d);
            }
        }
    }
    // Scales that are not finite become 0; whether there were any.
    __device__ __forceinline__ bool drop_odd() {
        bool odd = false;
#pragma unroll
        for (int si = 0; si < S::N; si++)
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (odd_scale(scale[si][i])) {
                    scale[si][i] = (f16)0.0f;
                    odd = true;
                }
        return odd;
    }
};

// What a query row sees: the slots below vis, and in a tree those of `mask` from base on.
struct Sees {
    uint32_t vis, base;
    uint64_t mask;
    __device__ __forceinline__ bool at(uint32_t slot) const {
        const uint32_t j = slot - base;
        return (slot < vis) | ((uint32_t)(mask >> (j & 63)) & (uint32_t)(j < 64));
    }
};

// Of row r of an item (end: of its farthest list).
__device__ __forceinline__ Sees sees(const Q4Params& p, const Q4Item& it, uint32_t r, bool valid, uint32_t end) {
    Sees s{valid ? it.base + (p.tree ? 0 : r) : end, it.base, 0};
    if (p.tree && valid) {
        const uint32_t row = it.row0 + r, named = end - it.base;
        s.mask = p.masks[2 * row] | (uint64_t)p.masks[2 * row + 1] << 32;
        if (named < 64) s.mask &= (1ull << named) - 1;
    }
    return s;
}

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
    return __builtin_amdgcn_readfirstlane((uint32_t)min((uint64_t)it.base + top, p.slot_limit));
}

// A row's scores are c s (c a power of two), its weights 2^(c s - ref). Where some score of these
// 32 slots passes ref by more than Q4_MOST, the refs rise to Q4_BIAS under their rows' maxima (to
// the maxima themselves where those are so large that the difference would be lost), and what
// was summed against the old one is to be multiplied by f.
__device__ __forceinline__ bool raise(const f32x4 (&s)[2], float c, float& ref, float& f) {
    float top = larger(larger(larger(s[0][0], s[0][1]), larger(s[0][2], s[0][3])),
                       larger(larger(s[1][0], s[1][1]), larger(s[1][2], s[1][3]))) * c;
    if (!__any(top > ref + Q4_MOST)) return false;
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    const float to = fmaxf(ref, fabsf(top) < 0x1p23f ? top - Q4_BIAS : top);
    f = to == -INFINITY ? 1.0f : exp2_hw(ref - to);
    ref = to;
    return true;
}

// The weights' B operand, the rounded values (hi) and the rest (lo); their sum goes to l. With
// PART, hi comes back as the rounded values times 1 - keep plus the rest times keep (0 or 1): a
// lane holds one part.
template <bool PART>
__device__ __forceinline__ void weights(const f32x4 (&s)[2], float c, float ref, float keep, float& l, half8& hi, half8& lo) {
    const float base = ref == -INFINITY ? 0.0f : ref;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const float w0 = exp2_hw(__builtin_fmaf(s[i >> 2][i & 3], c, -base));
        const float w1 = exp2_hw(__builtin_fmaf(s[i >> 2][(i & 3) + 1], c, -base));
        l += w0;
        l += w1;
        const half2 h = __builtin_convertvector((f32x2{w0, w1}), half2);
        const float k = PART ? -keep : -1.0f;
        const half2 r = __builtin_convertvector((f32x2{__builtin_fmaf((float)h[0], k, w0), __builtin_fmaf((float)h[1], k, w1)}), half2);
        hi[i] = PART ? r[0] : h[0];
        hi[i + 1] = PART ? r[1] : h[1];
        lo[i] = r[0];
        lo[i + 1] = r[1];
    }
}

__device__ __forceinline__ float ror8(float x) {  // lane n of each 16 gets lane (n + 8) % 16's
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x128, 0xf, 0xf, false));
}

constexpr uint32_t Q4_TILE = 32;

// Bytes of `slots` slots from the start of their first unit (rem elements into it).
__device__ __forceinline__ uint64_t q4_bytes(uint64_t slots, uint32_t rem, uint32_t kvd) {
    return (slots * kvd + rem + Q4_UNIT - 1) / Q4_UNIT * Q4_UNIT_BYTES;
}

// What bounds it, measured at 32 x 8 heads of 128, calls one after another over four layers' caches. Long
// lists: a tile is some 300 vector instructions a wave, most of them unpacking, against 256 cycles of MFMA;
// at 131072 slots the arithmetic alone takes 25 us and the loads alone 25, and two waves a SIMD overlap
// them to 41 (3.7 TB/s; the call 45). At 32768 slots 14.6 (the call 17.5; 19.7 where other caches come in
// between and nothing of these is left in the memory-side cache). Short ones: the chain from the launch over
// q, the first tile and the states to the result, 6.8 us at 1000 slots. Tried: two tiles on their way to a wave
// instead of one (15.1 us for 14.5 at 32768, and spills for heads past 160); operands read from memory where
// the lanes need them (1.6 times the time a tile); three waves a SIMD, the most that 155 registers allow
// (768 workgroups: 42.0 us at 131072 and the call 47.0, the states half as many again; 1024 are a second
// round for the last 256: 43.5 and 47.7).
template <int NB, bool PK, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void attn_q4_row(const Q4Params p) {
    constexpr int HD = 32 * NB, NF = 2 * NB, QW = NB < WAVES ? NB : WAVES, QJ = (NB + WAVES - 1) / WAVES;
    using S = Seg<NB>;
    using B = Raw<NB, Q4_TILE, 64>;
    __shared__ __attribute__((aligned(16))) union {
        uint8_t raw[WAVES][2][B::BYTES];
        f32x4 o[WAVES > 4 ? WAVES / 2 : 4][NF][64];
    } sh;
    __shared__ half8 sq[PK ? 1 : 2][NB][64];
    __shared__ float stop[QW][16], sr[WAVES][64], sl[WAVES][64];
    const Q4Bits bits;
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t m16 = lane & 15, g = lane >> 4;

    uint32_t ii = 0;
    if (p.nitems > 1) {  // the last item whose first block is at most this one
        const bool before = lane < p.nitems && p.items[lane].block0 <= blockIdx.z;
        ii = __builtin_amdgcn_readfirstlane(__popcll(__ballot(before)) - 1);
    }
    const Q4Item& it = p.items[ii];
    // Blocks 8 apart (one XCD) take the KV heads of one chunk: their bytes share cache lines.
    const uint32_t kvh = blockIdx.y, chunk = (blockIdx.z - it.block0) * 8 + ((blockIdx.x - it.turn) & 7);
    if (chunk >= it.nchunk) return;
    const uint32_t kvd = p.nkv * HD, nq = it.rows * p.G, end = p.tree ? tree_end(p, it) : it.base + it.rows - 1;
    const uint32_t all = (uint32_t)(((uint64_t)end + Q4_TILE - 1) / Q4_TILE), first = chunk * it.chunk;
    const uint32_t tiles = first < all ? min(it.chunk, all - first) : 0;

    // The chunk's bytes, from its first slot's unit to the end of the list.
    const uint64_t e0 = it.kvoff * kvd;
    const uint32_t rem0 = (uint32_t)(e0 & 255), rem = rem0 + kvh * HD;
    const uint64_t base = (e0 >> 8) * Q4_UNIT_BYTES, tile_bytes = (uint64_t)kvd * 18;
    const uint64_t from = base + first * tile_bytes, to = base + q4_bytes(end, rem0, kvd);
    // q's operands, each wave some of the steps for all; q's rows and the first tile are asked for together.
    const uint32_t n = PK ? (m16 & 7) : m16, r = (n * (65536 / p.G + 1)) >> 16;  // n / G
    const bool valid = n < nq;
    const uint32_t row = it.row0 + (valid ? r : 0), head = kvh * p.G + (valid ? n - r * p.G : 0);
    const Sees see = sees(p, it, r, valid, end);
    const size_t qrow = ((size_t)row * p.nh + head) * HD;
    float x[QJ][8], top = 0.0f;
#pragma unroll
    for (int i = 0; i < QJ; i++) q_load(p.q + qrow + 8 * (NB * g + i * WAVES + wave), valid && i * WAVES + wave < NB, x[i]);
    B kraw, vraw;
    kraw.set(rem, kvd, lane);
    vraw.set(rem, kvd, lane);
    auto load = [&](uint32_t t) {
        const uint64_t at = from + t * tile_bytes;
        kraw.load(q4_from(p.kc, at, to), kvd);
        vraw.load(q4_from(p.vc, at, to), kvd);
    };
    if (wave < tiles) load(wave);
#pragma unroll
    for (int i = 0; i < QJ; i++) top = q_top(x[i], top);
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    if (wave < QW && lane < 16) stop[wave][lane] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < QW; w++) top = fmaxf(top, stop[w][m16]);
    float k, c;
    q_scale(top, p.sc, k, c);
    const float keep = PK && m16 >= 8 ? 1.0f : 0.0f;
#pragma unroll
    for (int i = 0; i < QJ; i++) {
        const uint32_t j = i * WAVES + wave;
        if (j < NB) {
            half8 hi, lo;
            q_parts(x[i], k, hi, lo);
            if constexpr (PK) {
                sq[0][j][lane] = m16 < 8 ? hi : lo;
            } else {
                sq[0][j][lane] = hi;
                sq[1][j][lane] = lo;
            }
        }
    }
    __syncthreads();
    half8 qa[NB], qb[NB];
#pragma unroll
    for (int j = 0; j < NB; j++) {
        qa[j] = sq[0][j][lane];
        if constexpr (!PK) qb[j] = sq[1][j][lane];
    }

    f32x4 o[NF];
#pragma unroll
    for (int f = 0; f < NF; f++) o[f] = f32x4{0, 0, 0, 0};
    float ref = -INFINITY, l = 0.0f;

    for (uint32_t t = wave; t < tiles; t += WAVES) {
        const uint32_t ts = (first + t) * Q4_TILE;
        // The tile's bytes are the wave's own, and LDS serves a wave in order: its lanes' writes come
        // after their reads of the tile before and before those of this one.
        uint8_t *kt = sh.raw[wave][0], *vt = sh.raw[wave][1];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        kraw.store(kt);
        vraw.store(vt);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (t + WAVES < tiles) load(t + WAVES);
        f32x4 s[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}}, s2[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
        uint32_t kw[2][NB];
        f16 ks[2][NB];
#pragma unroll
        for (int h = 0; h < 2; h++) read_k<NB>(kt + (16 * h + m16) * B::SLOT, g, kw[h], ks[h]);
#pragma unroll
        for (int j = 0; j < NB; j++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const half8 a = unpack_k(bits, kw[h][j], ks[h][j]);
                s[h] = mfma16(a, qa[j], s[h]);
                if constexpr (!PK) s2[h] = mfma16(a, qb[j], s2[h]);
            }
        VRead<NB, false> v;
        v.read(vt, m16, g, 0);
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int i = 0; i < 4; i++) s[h][i] += PK ? ror8(s[h][i]) : s2[h][i];
        // A tile that some row does not see whole: scores of unseen slots become -inf, and V
        // scales that are not finite 0, their blocks put back as NaN for the rows that see them.
        const bool edge = ts + Q4_TILE > it.base;
        bool odd = false;
        if (edge) {
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (!see.at(ts + 16 * (i >> 2) + 4 * g + (i & 3))) s[i >> 2][i & 3] = -INFINITY;
            odd = v.drop_odd();
        }
        float f;
        if (raise(s, c, ref, f)) {
            l *= f;
#pragma unroll
            for (int i = 0; i < NF; i++) o[i] *= f;
        }
        half8 ph, pl;
        weights<PK>(s, c, ref, keep, l, ph, pl);
        auto pv = [&](auto width, int si) {
            constexpr int W = decltype(width)::value;
            half8 vf[W];
            unpack_v<W>(bits, v.word[si], v.scale[si], vf);
#pragma unroll
            for (int i = 0; i < W; i++) o[S::frag(si) + i] = mfma16(vf[i], ph, o[S::frag(si) + i]);
            if constexpr (!PK) {
#pragma unroll
                for (int i = 0; i < W; i++) o[S::frag(si) + i] = mfma16(vf[i], pl, o[S::frag(si) + i]);
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
                const bool seen = see.at(ts + i);
#pragma unroll
                for (int si = 0; si < S::N; si++) {  // (a lane's columns of a segment lie in one block)
                    const f16 d = *(const f16*)(vt + i * B::SLOT + 16 * NB + (S::col(si) + S::w(si) * 4 * g) / 32 * 2);
                    if (seen && odd_scale(d))
#pragma unroll
                        for (int w = 0; w < S::w(si); w++) o[S::frag(si) + w] = f32x4{NAN, NAN, NAN, NAN};
                }
            }
        }
    }

    // The waves' states, lane by lane: the upper half of more than four to the lower, then each of
    // four waves brings some of the columns together.
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
            for (int f = 0; f < NF; f++) sh.o[wave - half][f][lane] = o[f];
        }
        __syncthreads();
        if (wave < half) {
            const float other = sr[wave + half][lane], to = fmaxf(ref, other), ts = to == -INFINITY ? 0.0f : to;
            const float a = exp2_hw(ref - ts), e = exp2_hw(other - ts);
            l = l * a + sl[wave + half][lane] * e;
#pragma unroll
            for (int f = 0; f < NF; f++) o[f] = o[f] * a + sh.o[wave][f][lane] * e;
            ref = to;
        }
    }
    __syncthreads();
    if (wave < 4) {
        sr[wave][lane] = ref;
        sl[wave][lane] = l;
#pragma unroll
        for (int f = 0; f < NF; f++) sh.o[wave][f][lane] = o[f];
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
    const size_t unit = it.unit0 + kvh * it.nchunk + chunk;
    const float inv = it.nchunk > 1 ? 1.0f : L == 0.0f ? 0.0f : 1.0f / L;  // (a row that sees nothing: zeros)
    if (it.nchunk > 1 && wave == 0 && g == 0) *(float2*)(p.part_ml + 2 * (unit * 16 + n)) = float2{R, L};
    for (uint32_t f = wave; f < NF; f += 4) {
        f32x4 v = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < 4; w++) v += sh.o[w][f][lane] * a[w];
        v *= inv;
        if (it.nchunk > 1) {
            *(f32x4*)(p.part_o + ((unit * NF + f) * 64 + lane) * 4) = v;
        } else {
            const uint32_t col = column<NB>(f, g), step = stride<NB>(f);
#pragma unroll
            for (int i = 0; i < 4; i++) p.out[qrow + col + i * step] = v[i];
        }
    }
}

constexpr int Q4_WAVES = 4;

// More query rows: a tile of 64 slots unpacked once into LDS for the workgroup's waves of 16 RT
// query rows each: four of 32 rows, or eight of 16, of which four take each half of the slots.
//
// What bounds it. Prompts: the matrix cores, which q's and the weights' two parts give twice the work:
// 4096 rows of 32 x 8 heads of 128 take 272 to 278 us in a row of calls, 283 with other inputs in between: 485 to
// 505 TFLOP/s of the 549 that half of a large f16 product's rate leaves. Verify passes: latency. 8 rows of 64
// x 8 heads at 5003 slots take 14.6 us (the call 18.6), of which the first
// tile's way in some 6, three tiles 0.85 each (two barriers a tile) and 7 MB of states 1.5; eight waves
// a workgroup instead of four took 2 us off, 32 rows a wave there would leave half of the waves idle.
constexpr uint32_t Q4_TILE_B = 64;

template <int NB, int RT>
__global__ __launch_bounds__(RT == 1 ? 512 : 256, 2) void attn_q4_tile(const Q4Params p) {
    constexpr int HD = 32 * NB, NF = 2 * NB, KS = RT == 1 ? 2 : 1;
    constexpr uint32_t QT = 64 * RT;
    constexpr bool CUT = RT == 1;  // lists may be cut (32 rows a wave are taken where every CU has work)
    using S = Seg<NB>;
    __shared__ struct {
        half8 k[2][4][NB][64], v[2][2][NF][64];
    } fr;
    static_assert(KS == 1 || sizeof fr >= sizeof(f32x4) * 4 * NF * 64, "the second waves' states");
    using R = Raw<NB, Q4_TILE_B, 64 * Q4_WAVES>;
    __shared__ __attribute__((aligned(16))) uint8_t raw[2][R::BYTES];
    __shared__ uint32_t odd_tile[2];  // 1 + the tile of each buffer that held a scale that is not finite
    const Q4Bits bits;
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((threadIdx.x >> 6) & 3);
    const uint32_t ks = __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);  // KS 2: the second four waves
    const uint32_t m16 = lane & 15, g = lane >> 4;
    const Q4Item& it = p.items[0];
    // The longest lists first.
    const uint32_t kvh = blockIdx.x, chunk = CUT ? blockIdx.y : 0, qt = p.nqt - 1 - blockIdx.z;
    const uint32_t kvd = p.nkv * HD, nq = it.rows * p.G, q0 = qt * QT, q1 = min(q0 + QT, nq);
    const uint32_t r0 = q0 / p.G, h0 = q0 - r0 * p.G;
    const uint32_t seen = p.tree ? it.base : it.base + r0;  // slots every row here sees
    const uint32_t end = p.tree ? tree_end(p, it) : it.base + (q1 - 1) / p.G;
    const uint32_t all = (uint32_t)(((uint64_t)end + Q4_TILE_B - 1) / Q4_TILE_B), t0 = chunk * it.chunk;
    const size_t unit = ((size_t)kvh * p.nqt + qt) * it.nchunk + chunk;
    // Nothing of these rows' lists. (Only cut ones get here; compiled for CUT alone, the other form's loop
    // is ordered another way and 4096 rows of 32 x 8 heads take 276 us, not 272.)
    if (t0 >= all && it.nchunk > 1) {
        if (threadIdx.x < QT) *(float2*)(p.part_ml + 2 * (unit * QT + threadIdx.x)) = float2{-INFINITY, 0.0f};
        return;
    }
    const uint32_t t1 = min(t0 + it.chunk, all);

    const uint64_t e0 = it.kvoff * kvd;
    const uint32_t rem0 = (uint32_t)(e0 & 255), rem = rem0 + kvh * HD;
    const uint64_t base = (e0 >> 8) * Q4_UNIT_BYTES, tile_bytes = (uint64_t)kvd * 36, to = base + q4_bytes(end, rem0, kvd);

    // q's rows and the first tile are asked for together.
    Sees see[RT];
    half8 qh[RT][NB], ql[RT][NB];
    float c[RT], x[RT][NB][8], top[RT];
#pragma unroll
    for (int r = 0; r < RT; r++) {
        const uint32_t i = (wave * RT + r) * 16 + m16, y = h0 + i, dr = (y * (65536 / p.G + 1)) >> 16;  // y / G
        const bool valid = q0 + i < nq;
        const uint32_t row = it.row0 + (valid ? r0 + dr : 0), head = kvh * p.G + (valid ? y - dr * p.G : 0);
        see[r] = sees(p, it, r0 + dr, valid, end);
        const float* q = p.q + ((size_t)row * p.nh + head) * HD;
        top[r] = 0.0f;
#pragma unroll
        for (int j = 0; j < NB; j++) q_load(q + 8 * (NB * g + j), valid, x[r][j]);
    }
    // (KS 2: four waves fetch and unpack K, four V.)
    R kraw, vraw;
    const uint32_t thread = threadIdx.x & 255;
    kraw.set(rem, kvd, thread);
    if constexpr (KS == 1) vraw.set(rem, kvd, thread);
    auto fetch = [&](uint32_t t) {
        const uint64_t at = base + t * tile_bytes;
        kraw.load(q4_from(KS == 2 && ks ? p.vc : p.kc, at, to), kvd);
        if constexpr (KS == 1) vraw.load(q4_from(p.vc, at, to), kvd);
    };
    auto store = [&]() {
        kraw.store(raw[KS == 2 ? ks : 0]);
        if constexpr (KS == 1) vraw.store(raw[1]);
    };
    if (t0 < t1) fetch(t0);
#pragma unroll
    for (int r = 0; r < RT; r++) {
        float k;
#pragma unroll
        for (int j = 0; j < NB; j++) top[r] = q_top(x[r][j], top[r]);
        top[r] = fmaxf(top[r], __shfl_xor(top[r], 16));
        top[r] = fmaxf(top[r], __shfl_xor(top[r], 32));
        q_scale(top[r], p.sc, k, c[r]);
#pragma unroll
        for (int j = 0; j < NB; j++) q_parts(x[r][j], k, qh[r][j], ql[r][j]);
    }

    // This wave's share of a tile's operands: K's of slots 16 wave .. + 15, and of V's of slots 32 step ..
    // + 31 half the columns of every lane.
    const uint32_t half = wave & 1, step = wave >> 1;
    auto unpack = [&](uint32_t t, int buf) {
        if (KS == 1 || ks == 0) {
            uint32_t kw[NB];
            f16 kd[NB];
            read_k<NB>(raw[0] + (16 * wave + m16) * R::SLOT, g, kw, kd);
#pragma unroll
            for (int j = 0; j < NB; j++) fr.k[buf][wave][j][lane] = unpack_k(bits, kw[j], kd[j]);
        }
        if (KS == 2 && ks == 0) return;
        VRead<NB, true> v;
        v.read(raw[1] + 32 * step * R::SLOT, m16, g, half);
        if (t * Q4_TILE_B + Q4_TILE_B > seen && v.drop_odd()) odd_tile[buf] = t + 1;  // some row does not see all of it
#pragma unroll
        for (int si = 0; si < S::N; si++) {
            if (S::w(si) == 8) {
                half8 x[4];
                unpack_v<4>(bits, v.word[si], v.scale[si], x);
#pragma unroll
                for (int k = 0; k < 4; k++) fr.v[buf][step][S::frag(si) + 4 * half + k][lane] = x[k];
            } else if (S::w(si) == 4) {
                half8 x[2];
                unpack_v<2>(bits, v.word[si], v.scale[si], x);
#pragma unroll
                for (int k = 0; k < 2; k++) fr.v[buf][step][S::frag(si) + 2 * half + k][lane] = x[k];
            } else {
                half8 x[2];
                unpack_v<2>(bits, v.word[si], v.scale[si], x);
                fr.v[buf][step][S::frag(si) + half][lane] = half ? x[1] : x[0];
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
    if (t0 < t1) store();
    __syncthreads();
    if (t0 < t1) {
        if (t0 + 1 < t1) fetch(t0 + 1);
        unpack(t0, 0);
    }
    __syncthreads();
    for (uint32_t t = t0; t < t1; t++) {
        const int buf = (t - t0) & 1;
        const uint32_t ts = t * Q4_TILE_B;
        if (t + 1 < t1) {  // the next tile's bytes, unpacked behind this tile's products
            store();
            __syncthreads();
            if (t + 2 < t1) fetch(t + 2);
        }
        const bool edge = ts + Q4_TILE_B > seen;
#pragma unroll
        for (int i = 0; i < 2 / KS; i++) {
            const uint32_t u = KS == 2 ? ks : i;  // 32 of the tile's slots
            // (Four sums in turn, so that no MFMA waits for the one before: one set of rows takes the
            // parts of q apart.)
            constexpr int LO = RT == 1 ? 1 : 0;
            f32x4 s[RT][2], s2[2];
#pragma unroll
            for (int r = 0; r < RT; r++) s[r][0] = s[r][1] = s2[0] = s2[1] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < NB; j++) {
                const half8 k0 = fr.k[buf][2 * u][j][lane], k1 = fr.k[buf][2 * u + 1][j][lane];
#pragma unroll
                for (int r = 0; r < RT; r++) {
                    s[r][0] = mfma16(k0, qh[r][j], s[r][0]);
                    s[r][1] = mfma16(k1, qh[r][j], s[r][1]);
                }
#pragma unroll
                for (int r = 0; r < RT; r++) {
                    f32x4(&to)[2] = LO ? s2 : s[r];
                    to[0] = mfma16(k0, ql[r][j], to[0]);
                    to[1] = mfma16(k1, ql[r][j], to[1]);
                }
            }
            half8 ph[RT], pl[RT];
#pragma unroll
            for (int r = 0; r < RT; r++) {
                if (LO) {
                    s[r][0] += s2[0];
                    s[r][1] += s2[1];
                }
                if (edge)
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        if (!see[r].at(ts + 32 * u + 16 * (i >> 2) + 4 * g + (i & 3))) s[r][i >> 2][i & 3] = -INFINITY;
                float f;
                if (raise(s[r], c[r], ref[r], f)) {
                    l[r] *= f;
#pragma unroll
                    for (int k = 0; k < NF; k++) o[r][k] *= f;
                }
                weights<false>(s[r], c[r], ref[r], 0.0f, l[r], ph[r], pl[r]);
            }
#pragma unroll
            for (int f = 0; f < NF; f += 2) {
                const half8 v0 = fr.v[buf][u][f][lane], v1 = fr.v[buf][u][f + 1][lane];
#pragma unroll
                for (int r = 0; r < RT; r++) {
                    o[r][f] = mfma16(v0, ph[r], o[r][f]);
                    o[r][f + 1] = mfma16(v1, ph[r], o[r][f + 1]);
                }
#pragma unroll
                for (int r = 0; r < RT; r++) {
                    o[r][f] = mfma16(v0, pl[r], o[r][f]);
                    o[r][f + 1] = mfma16(v1, pl[r], o[r][f + 1]);
                }
            }
        }
        if (edge && odd_tile[buf] == t + 1) {
            const q4_rsrc vr = q4_from(p.vc, base + t * tile_bytes, to);
            for (uint32_t i = 0; i < Q4_TILE_B && ts + i < end; i++)
#pragma unroll
                for (int si = 0; si < S::N; si++) {
                    const bool odd = odd_scale(load_scale(vr, q4_scale_at32(rem + i * kvd + S::col(si) + S::w(si) * 4 * g)));
#pragma unroll
                    for (int r = 0; r < RT; r++)
                        if (odd && see[r].at(ts + i))
#pragma unroll
                            for (int k = 0; k < S::w(si); k++) o[r][S::frag(si) + k] = f32x4{NAN, NAN, NAN, NAN};
                }
        }
        if (t + 1 < t1) unpack(t + 1, buf ^ 1);
        __syncthreads();
    }

    if constexpr (KS == 2) {  // the two halves of the slots
        f32x4(*so)[NF][64] = (f32x4(*)[NF][64])&fr;
        float(*sr)[2][64] = (float(*)[2][64])raw;
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
        const uint32_t sl = (wave * RT + r) * 16 + m16;
        if (q0 + sl >= nq) continue;
        if (CUT && it.nchunk > 1) {
            f32x4* part = (f32x4*)p.part_o + (unit * (QT / 16) + sl / 16) * NF * 64 + lane;
#pragma unroll
            for (int f = 0; f < NF; f++) part[64 * f] = o[r][f];
            if (g == 0) *(float2*)(p.part_ml + 2 * (unit * QT + sl)) = float2{ref[r], l[r]};
            continue;
        }
        const uint32_t y = h0 + sl, dr = (y * (65536 / p.G + 1)) >> 16;
        float* dst = p.out + ((size_t)(it.row0 + r0 + dr) * p.nh + kvh * p.G + y - dr * p.G) * HD;
        const float k = l[r] == 0.0f ? 0.0f : 1.0f / l[r];
#pragma unroll
        for (int si = 0; si < S::N; si++)
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int x = 0; x < S::w(si); x++)
                    dst[S::col(si) + S::w(si) * (4 * g + i) + x] = o[r][S::frag(si) + x][i] * k;
    }
}

// The chunks of 16 query rows of a list brought together, one operand's columns a workgroup (two took
// 0.4 to 1.9 us more, few workgroups reading much each), each wave a share of the chunks; states lie as
// their waves held them: 3 to 4 us of a call, a launch behind the other kernel and one read of the states.
// A chunk without a weight left
// its columns unwritten.
constexpr uint32_t Q4_MAX_CHUNKS = 256;

template <int NB, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void attn_q4_fold(const Q4Params p) {
    constexpr int HD = 32 * NB, NF = 2 * NB, AHEAD = 8;
    __shared__ f32x4 sum[WAVES][64];
    __shared__ float sr[WAVES][64], sl[WAVES][64];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m16 = lane & 15, g = lane >> 4;
    const uint32_t f = blockIdx.x, kvh = blockIdx.y, z = blockIdx.z;
    const Q4Item& it = p.items[p.nitems > 1 ? z : 0];
    const uint32_t chunks = it.nchunk;
    if (chunks == 1) return;  // written by its workgroup
    const uint32_t n0 = p.nitems > 1 ? 0 : 16 * z, n = n0 + m16, sl0 = n0 & (p.qt - 1);  // this row of the item's
    const bool valid = n < it.rows * p.G;
    const size_t u0 = it.unit0 + ((size_t)kvh * p.nqt + n0 / p.qt) * chunks;
    const float2* ml = (const float2*)p.part_ml + u0 * p.qt + sl0 + m16;
    const f32x4* at = (const f32x4*)p.part_o + ((u0 * (p.qt / 16) + sl0 / 16) * NF + f) * 64 + lane;
    const size_t next = (size_t)(p.qt / 16) * NF * 64;
    f32x4 a = {0, 0, 0, 0};
    float R = -INFINITY, L = 0.0f;
    for (uint32_t c0 = wave; c0 < chunks; c0 += AHEAD * WAVES) {
        float2 s[AHEAD];
        f32x4 x[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            const uint32_t c = c0 + i * WAVES;
            const bool there = valid && c < chunks;
            s[i] = there ? ml[(size_t)c * p.qt] : float2{-INFINITY, 0.0f};
            x[i] = there ? at[c * next] : f32x4{0, 0, 0, 0};
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
    const float k = L == 0.0f ? 0.0f : 1.0f / L;
    const uint32_t r = n / p.G, step = stride<NB>(f);
    float* dst = p.out + ((size_t)(it.row0 + r) * p.nh + kvh * p.G + n - r * p.G) * HD + column<NB>(f, g);
#pragma unroll
    for (int i = 0; i < 4; i++) dst[i * step] = a[i] * k;
}

template <int NB, int WAVES>
void launch_row(const Q4Params& p, uint32_t octs, bool pk, const AttnCall& a, hipStream_t s) {
    const dim3 grid(8, p.nkv, octs), wg(64 * WAVES);
    // (Eight waves have 256 registers a lane; more than eight query rows of heads past 192 want more.)
    constexpr int W = NB > 6 ? Q4_WAVES : WAVES;
    if (pk) hipExtLaunchKernelGGL((attn_q4_row<NB, true, WAVES>), grid, wg, 0, s, a.ev_before, a.ev_after, 0, p);
    else hipExtLaunchKernelGGL((attn_q4_row<NB, false, W>), grid, dim3(64 * W), 0, s, a.ev_before, a.ev_after, 0, p);
}
template <int NB>
void launch_tile(const Q4Params& p, uint32_t rt, const AttnCall& a, hipStream_t s) {
    const dim3 grid(p.nkv, p.items[0].nchunk, p.nqt);
    if constexpr (NB <= 4) {
        if (rt == 2) {
            hipExtLaunchKernelGGL((attn_q4_tile<NB, 2>), grid, dim3(256), 0, s, a.ev_before, a.ev_after, 0, p);
            return;
        }
    }
    hipExtLaunchKernelGGL((attn_q4_tile<NB, 1>), grid, dim3(512), 0, s, a.ev_before, a.ev_after, 0, p);
}
template <int NB>
void launch_fold(const Q4Params& p, uint32_t groups, hipStream_t s) {
    // A wave alone holds a few chunks' states at once; more chunks are shared out.
    uint32_t most = 0;
    for (uint32_t i = 0; i < p.nitems; i++) most = std::max(most, p.items[i].nchunk);
    const dim3 grid(2 * NB, p.nkv, groups);
    if (most <= 8) hipLaunchKernelGGL((attn_q4_fold<NB, 1>), grid, dim3(64), 0, s, p);
    else hipLaunchKernelGGL((attn_q4_fold<NB, 8>), grid, dim3(512), 0, s, p);
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

// Workgroups of attn_q4_row that keep the GPU busy without more states than they are worth: two a CU (a
// step of 32 x 8 heads of 128 at 131072 slots: 45.5 us at 512 and at 256, 47.0 at 768, 47.7 at 1024; at 32768
// 17.5 at 512, which Q4_FOLD_CHUNKS holds it to, 17.0 at 256).
constexpr uint32_t Q4_ROW_GROUPS = 512;
// Lists of several lengths end at different times: more workgroups (16 of 28 x 4 heads of 128 at 1 to 16384
// slots: 38 us at 768, 46 at 512, 40 at 1024).
constexpr uint32_t Q4_RAGGED_GROUPS = 768;
// Tiles of a list up to which one workgroup of eight waves takes it whole, without a second launch
// (32 x 8 heads of 128: 8.0 us at 16 tiles against 9.4, 11.3 at 32 against 10). Of several lists their
// average, if the longest has at most twice that (8 lists of 28 x 4 heads, one of 1500 slots and the
// rest of 200: 9.8 us cut, 13.4 whole).
constexpr uint32_t Q4_BRIEF = 20;

// Chunks that attn_q4_fold reads at once, and the tiles a chunk past them is worth (28 x 4 heads of 128 at
// 24000 slots: 12.5 us in 63 chunks, 14.7 in 94).
constexpr uint32_t Q4_FOLD_CHUNKS = 64, Q4_FOLD_TILES = 16;

// Chunks for a list of `tiles` tiles, `least` at least a chunk, for `want` of them; of multiples of `of` (a
// chunk of attn_q4_row takes as long as its first wave, so fewer chunks of whole rounds: 9.6 us for 10.2 at
// 1300 slots of 32 x 8 heads).
void cut(Q4Item& it, uint64_t tiles, uint32_t want, uint32_t least, uint32_t of) {
    const uint64_t n = std::max<uint64_t>(1, std::min<uint64_t>({(uint64_t)want, tiles / least, std::max<uint64_t>(Q4_FOLD_CHUNKS, tiles / Q4_FOLD_TILES), Q4_MAX_CHUNKS}));
    it.chunk = (uint32_t)std::max<uint64_t>(1, ((tiles + n - 1) / n + of - 1) / of * of);
    it.nchunk = (uint32_t)std::max<uint64_t>(1, (tiles + it.chunk - 1) / it.chunk);
}

// Chunks of attn_q4_tile's lists of `tiles` tiles for `units` workgroups a chunk: those of the least time
// by what was measured (us): 0.6 + 0.006 hd a tile and 7 a workgroup beside, one at a time a CU; for
// a second launch 2 + 0.0006 hd a unit, and the states' write and read at 5 TB/s. So 200 rows of 32 x 8 heads of
// 128 run whole at 300 slots (18 us, in two chunks 25) and in two at 4000 (63, whole 96, in four 68), 340 rows at
// 16000 in four (288, whole 352, in two 367), 8 rows of 64 x 8 at 500 in four (12.5, whole 17.5).
uint32_t tile_chunks(uint64_t tiles, uint64_t units, uint32_t hd) {
    constexpr uint64_t CUS = 256;
    const float tile = 0.6f + 0.006f * hd, launch = 2.0f + 0.0006f * hd * units, states = 64.0f * 8.0f / 5e6f * hd * units;
    uint64_t best = 1;
    float least = (float)((units + CUS - 1) / CUS) * (tile * tiles + 7.0f);
    for (uint64_t half = 1; half <= 8; half++) {  // as many as half a round holds, one round, ... four
        const uint64_t n = std::min<uint64_t>({CUS * half / 2 / units, tiles / 2, Q4_MAX_CHUNKS});
        if (n < 2) continue;
        const float t = (float)((units * n + CUS - 1) / CUS) * (tile * ((tiles + n - 1) / n) + 7.0f) + launch + states * n;
        if (t < least) least = t, best = n;
    }
    return (uint32_t)best;
}

bool reserve(Q4Params& p, uint64_t states, uint32_t hd, Workspace& ws) {
    const bool had = ws.reserve_if(states, hd <= 32 ? 32 : hd <= 64 ? 64 : hd <= 128 ? 128 : 256);
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
    uint64_t total = 0, most = 0;
    for (uint32_t i = 0; i < p.nitems; i++) {
        const uint64_t tiles = (lens[i] + Q4_TILE - 1) / Q4_TILE;
        total += tiles;
        most = std::max(most, tiles);
    }
    const uint32_t want = std::max(1u, (p.nitems > 1 ? Q4_RAGGED_GROUPS : Q4_ROW_GROUPS) / a.nkv);
    uint32_t units, octs;
    bool split;
    auto plan = [&](uint64_t all) {
        units = octs = 0;
        split = false;
        for (uint32_t i = 0; i < p.nitems; i++) {
            Q4Item& it = p.items[i];
            const uint64_t tiles = (lens[i] + Q4_TILE - 1) / Q4_TILE;
            it.unit0 = units;
            it.block0 = octs;
            it.turn = units / a.nkv % 8;
            // A list's share of the workgroups is its share of the tiles.
            cut(it, tiles, (uint32_t)std::max<uint64_t>(1, all * tiles / std::max<uint64_t>(1, total)), Q4_WAVES, Q4_WAVES);
            units += it.nchunk * a.nkv;
            octs += (it.nchunk + 7) / 8;
            split |= it.nchunk > 1;
        }
    };
    // Lists that eight waves take in a few tiles each are not cut: no second launch.
    const bool brief = total <= (uint64_t)p.nitems * Q4_BRIEF && most <= 2 * Q4_BRIEF;
    plan(brief ? 0 : want);
    if (split && !reserve(p, (uint64_t)units * 16, a.hd, ws)) plan(0);
    const bool pk = p.items[0].rows * p.G <= 8;
#define Q4_BRIEF_ROW(NB) launch_row<NB, 2 * Q4_WAVES>(p, octs, pk, a, s)
#define Q4_ROW(NB) launch_row<NB, Q4_WAVES>(p, octs, pk, a, s)
    if (brief) {
        Q4_BY_DIM(a.hd / 32, Q4_BRIEF_ROW)
    } else {
        Q4_BY_DIM(a.hd / 32, Q4_ROW)
    }
#undef Q4_ROW
#undef Q4_BRIEF_ROW
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || !split) return e;
#define Q4_FOLD(NB) launch_fold<NB>(p, p.nitems, s)
    Q4_BY_DIM(a.hd / 32, Q4_FOLD)
#undef Q4_FOLD
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
    const uint32_t most = 65535 * 64 / p.G;  // rows whose units of query rows a grid holds
    if (a.rows > most) {
        AttnCall part = a;
        for (uint32_t r = 0; r < a.rows; r += most) {
            part.rows = std::min(most, a.rows - r);
            part.pos = a.pos + r;
            part.q = a.q + (size_t)r * a.nh * a.hd;
            part.out = a.out + (size_t)r * a.nh * a.hd;
            const hipError_t e = q4_attention(part, ws, s);
            if (e != hipSuccess) return e;
            part.ev_before = part.ev_after = nullptr;
        }
        return hipSuccess;
    }
    // 32 query rows a wave halve the LDS reads a product, where enough such workgroups keep every CU busy
    // (32 x 8 heads of 128, 4096 rows, in a row of calls: 272 us, 397 with 16; 1000 rows: 51, 39 with 16; they meet at 1300.
    // Heads of 64 read less: 14 x 2 of them, 4096 rows, 124 us and 100 with 16, 8192 rows 314 and 329).
    const uint32_t rt = a.hd <= 128 && (nq + 127) / 128 * a.nkv >= (a.hd > 64 ? 352u : 768u) ? 2 : 1;
    p.qt = 64 * rt;
    p.nqt = (uint32_t)((nq + p.qt - 1) / p.qt);
    const uint64_t groups = (uint64_t)p.nqt * a.nkv, tiles = (far + Q4_TILE_B - 1) / Q4_TILE_B;
    // (attn_q4_tile<., 2> knows whole lists only.)
    cut(it, tiles, rt == 2 ? 1 : tile_chunks(tiles, groups, a.hd), 2, 1);
    if (it.nchunk > 1 && !reserve(p, groups * it.nchunk * p.qt, a.hd, ws)) cut(it, tiles, 1, 2, 1);
#define Q4_TILES(NB) launch_tile<NB>(p, rt, a, s)
    Q4_BY_DIM(a.hd / 32, Q4_TILES)
#undef Q4_TILES
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || it.nchunk == 1) return e;
#define Q4_FOLD(NB) launch_fold<NB>(p, (uint32_t)((nq + 15) / 16), s)
    Q4_BY_DIM(a.hd / 32, Q4_FOLD)
#undef Q4_FOLD
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
