// A KV cache in pages: the parameters of the kernels that attend over it, and how they bring tiles of
// it into LDS.
//
// A pool's K and V are [pages][page slots][kvd]; slot t of sequence i is slot t % page slots of page
// table[i][t / page slots]. Pages are powers of two of at least 16 slots, so the 16 slots of a granule
// lie in one page, one after another: a granule is one buffer descriptor, which ends with the list's
// last slot (what is asked for past that comes back as zeros, whatever a reused page holds there) and
// is empty for a page number past the pool.
//
// Granules go to LDS by buffer loads that write LDS themselves, 64 lanes x 16 bytes in a row: a slot's
// bytes follow each other at PITCH, its 16-byte units turned by an amount of its own so that the reads
// of 16 slots' units at once meet all banks. The loads are inline asm without outputs: the compiler
// would else wait for all of them before every transposing read, not knowing which tile that reads.
// Whoever reads waits by wait_loads (and a barrier, for other waves' loads) first.
#pragma once

#include "common.hpp"

namespace bchip {

// A sequence's new rows (q and out rows row0 ..) over its `len` slots, which end with theirs: row r sees
// the slots below len - rows + r + 1. block0: the first of its blocks of its kind in the launch; fold0: of
// its groups of 16 query rows in the fold's.
struct PgItem {
    uint32_t row0, len, rows_seq, block0, fold0;  // rows << 8 | sequence (its line of the table)
};

constexpr uint32_t PG_ITEMS = 128;  // of a launch: two a lane

// Items are of two kinds: the first nrow have at most 16 query rows (attn_paged_row's), the others more
// (attn_paged_tile16's or 32's).
struct PgParams {
    const float* q;
    const uint8_t* kc;
    const uint8_t* vc;
    float* out;
    float* part_o;   // chunk states [item, KV head, 16 query rows, chunk][HD / 16][64][4]
    float* part_ml;  // [...][16][2]: their references and sums
    const uint32_t* pages;
    uint32_t page_stride, page_shift, npages;
    uint32_t nh, nkv, hd, G;
    float sc;                 // scale * log2(e)
    uint32_t chunk, tchunk;   // tiles a chunk, of either kind
    uint32_t blocks, tblocks; // blocks / KV heads
    uint32_t qt;              // query rows a block of the second kind, whose states lie behind the first's
    uint32_t nrow, nitems;
    PgItem items[PG_ITEMS];
};

// The last of items lo .. hi - 1 whose first block (fold: group) is at most x.
template <bool FOLD>
__device__ __forceinline__ uint32_t item_of(const PgParams& p, uint32_t lo, uint32_t hi, uint32_t x) {
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t a = FOLD ? p.items[lane].fold0 : p.items[lane].block0, b = FOLD ? p.items[lane + 64].fold0 : p.items[lane + 64].block0;
    const uint32_t n = __popcll(__ballot(lane >= lo && lane < hi && a <= x)) + __popcll(__ballot(lane + 64 >= lo && lane + 64 < hi && b <= x));
    return __builtin_amdgcn_readfirstlane(lo + n - 1);
}

// A block's item and its number. Every argument that a kernel's first loads need is read here, item 0 with
// them, in one round trip: a branch that waits for one argument would else put the others' behind it (the
// empty asm is their use).
template <bool FOLD>
__device__ __forceinline__ PgItem item_with_arguments(const PgParams& p, bool rows, uint32_t x, uint32_t& which) {
    PgItem it = p.items[0];
    asm volatile("" ::"s"(p.q), "s"(p.kc), "s"(p.vc), "s"(p.out), "s"(p.part_o), "s"(p.part_ml), "s"(p.pages), "s"(p.page_stride),
                 "s"(p.page_shift), "s"(p.npages), "s"(p.nh), "s"(p.nkv), "s"(p.hd), "s"(p.G), "s"(p.sc), "s"(p.chunk), "s"(p.tchunk), "s"(p.qt),
                 "s"(p.blocks), "s"(p.nrow), "s"(p.nitems), "s"(it.row0), "s"(it.len), "s"(it.rows_seq), "s"(it.block0), "s"(it.fold0));
    which = 0;
    if (p.nitems > 1) {
        which = item_of<FOLD>(p, FOLD || rows ? 0 : p.nrow, !FOLD && rows ? p.nrow : p.nitems, x);
        it = p.items[which];
    }
    return it;
}

typedef uint32_t pg_u32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) uint8_t pg_lds;

// 64 lanes' 16 bytes at their offsets to LDS, one after another from `to` + `plus`, a constant once its loop is
// unrolled (sums made outside would each hold a scalar register, and there are not as many). A vector memory
// instruction may read a scalar that a vector one wrote (a spilled descriptor's v_readlane) five wait states
// later, and M0 one; the compiler counts neither for an asm block. The sum is one, s_nop 3 the other four.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // (M0 is one of its reserved registers: named so that it keeps no offset of its own there)
__device__ __forceinline__ void load_lds(pg_u32x4 from, uint32_t offset, uint32_t to, uint32_t plus) {
    asm volatile("s_add_u32 m0, %2, %3\n\ts_nop 3\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(offset), "s"(from), "s"(to), "i"(plus) : "memory", "m0", "scc");
}
#pragma clang diagnostic pop
// Until at most N of this wave's loads are on their way.
template <int N>
__device__ __forceinline__ void wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// This wave's reads and writes of LDS are done.
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// Granules of heads of 32 NB dims.
template <typename KVT, int NB>
struct PgTile {
    static constexpr int ES = sizeof(KVT), PITCH = 32 * NB * ES, UNITS = PITCH / 16, GRANULE = 16 * PITCH, LOADS = GRANULE / 1024;
    // Slots after which the units of a row start at the same bank again: 1 << (2 - SHIFT) ... of 16 units.
    static constexpr int SHIFT = UNITS % 16 == 0 ? 0 : UNITS % 8 == 0 ? 1 : 2;
    static __device__ __forceinline__ uint32_t turn_k(uint32_t slot) { return (slot & 15) >> SHIFT; }
    // (f16: a transposing read takes two units of each of eight slots at once; f32: a whole slot's.)
    static __device__ __forceinline__ uint32_t turn_v(uint32_t slot) { return ES == 2 ? 2 * ((slot & 7) >> SHIFT) : 0; }
    static __device__ __forceinline__ uint32_t at(uint32_t slot, uint32_t unit, uint32_t turn) {
        return slot * PITCH + (unit + turn) % UNITS * 16;
    }
    // Where in a granule (rows of row_bytes) this lane's bytes of load i come from; past the head: nowhere.
    template <bool V>
    static __device__ __forceinline__ uint32_t from(int i, uint32_t lane, uint32_t row_bytes, uint32_t head_bytes) {
        const uint32_t x = 64 * i + lane, slot = x / UNITS, turn = V ? turn_v(slot) : turn_k(slot);
        const uint32_t unit = (x % UNITS + UNITS - turn) % UNITS;
        return 16 * unit < head_bytes ? slot * row_bytes + 16 * unit : 0x80000000u;
    }
};

// A sequence's slots of one KV head.
struct PgList {
    const uint32_t* table;
    uint32_t end, shift, npages;
    uint32_t row_bytes, head;  // bytes of a slot, and of the heads before this one
    __device__ __forceinline__ uint32_t page(uint32_t slot) const {  // of a slot, or of the last one
        return ((const __attribute__((address_space(4))) uint32_t*)table)[min(slot, end - 1) >> shift];
    }
    __device__ __forceinline__ bool bad(uint32_t slot, uint32_t page) const { return slot < end && page >= npages; }
    // The granule from `slot` on (a multiple of 16), which lies in `page`: where it starts, its bytes.
    __device__ __forceinline__ uint64_t place(const uint8_t* cache, uint32_t slot, uint32_t page) const {
        return (uint64_t)cache + (((uint64_t)page << shift) + (slot & ((1u << shift) - 1))) * row_bytes + head;
    }
    __device__ __forceinline__ uint32_t size(uint32_t slot, uint32_t page) const {
        const uint32_t n = slot < end && page < npages ? min(16u, end - slot) : 0;
        return n ? n * row_bytes - head : 0u;
    }
    static __device__ __forceinline__ uint32_t same(uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); }
    __device__ __forceinline__ pg_u32x4 granule(const uint8_t* cache, uint32_t slot, uint32_t page) const {
        const uint64_t at = place(cache, slot, page);
        return pg_u32x4{same((uint32_t)at), same((uint32_t)(at >> 32) & 0xffffu), same(size(slot, page)), 0x00020000u};
    }
    // The same for loads into registers.
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const uint8_t* cache, uint32_t slot, uint32_t page) const {
        const uint64_t at = place(cache, slot, page);
        return __builtin_amdgcn_make_buffer_rsrc((void*)((uint64_t)same((uint32_t)(at >> 32)) << 32 | same((uint32_t)at)), 0, (int)same(size(slot, page)), 0x00020000);
    }
};

__device__ __forceinline__ PgList list_of(const PgParams& p, const PgItem& it, uint32_t kvh, uint32_t es) {
    return PgList{p.pages + (size_t)(it.rows_seq & 255) * p.page_stride, it.len, p.page_shift, p.npages, p.nkv * p.hd * es, kvh * p.hd * es};
}

// Lane i of 16 gets the i'th f16 of each of four rows that the sixteen lanes' addresses name, four
// lanes a row.
__device__ __forceinline__ half4 read_transposed(const uint8_t* at) {
    typedef int16_t s16x4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)at));
}

// One f32 product of 16 x 16 x 4: lane l holds A[l % 16][l / 16], B[l / 16][l % 16], D[4 (l / 16) + i][l % 16].
__device__ __forceinline__ f32x4 mfma_f32(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// Where result register i of lane group g of operand f lies in a head. f16: dims 16 f + 4 g + i. f32: the
// operands of a segment of 64 dims (four; of a last one of 32, two) take every fourth (second) of them.
template <typename KVT, int NB>
__device__ __forceinline__ uint32_t dim_of(uint32_t f, uint32_t g, uint32_t i) {
    if (sizeof(KVT) == 2) return 16 * f + 4 * g + i;
    const uint32_t s = f / 4;
    return 64 * s + (s < NB / 2 ? 4 : 2) * (4 * g + i) + f % 4;
}

__device__ __forceinline__ bool odd16(uint32_t pair) {  // either half an infinity or a NaN
    return (pair & 0x7c00u) == 0x7c00u || (pair & 0x7c000000u) == 0x7c000000u;
}
__device__ __forceinline__ bool odd32(uint32_t x) { return (x & 0x7f800000u) == 0x7f800000u; }

}  // namespace bchip
