// The launches of the kernels over pages, which live in files of their own.
#pragma once

#include "paged.hpp"

namespace bchip {

// Whether every item of the first kind has at most eight query rows.
inline bool pg_few(const PgParams& p) {
    for (uint32_t i = 0; i < p.nrow; i++)
        if ((p.items[i].rows_seq >> 8) * p.G > 8) return false;
    return true;
}
// Tiles of 32 slots (f16 caches) or 16 (f32).
constexpr uint32_t pg_row_tile(bool f16_cache) { return f16_cache ? 32 : 16; }
// brief: lists of few tiles, by eight waves each (heads past 128 dims: four).
void paged_rows_launch(const PgParams& p, bool f16_cache, bool brief, hipStream_t s);

// Tiles of 64 slots (f16) or 32 (f32); p.qt query rows a block: 128 (heads of up to 128 dims) or 64.
constexpr uint32_t pg_tile(bool f16_cache) { return f16_cache ? 64 : 32; }
void paged_tiles_launch(const PgParams& p, bool f16_cache, hipStream_t s);
// Both kinds in one launch: f32 caches, and f16 heads of up to 128 dims.
void paged_mixed_launch(const PgParams& p, bool f16_cache, hipStream_t s);
// The chunks of the items that have more than one (`most` at most), groups of 16 query rows of them.
void paged_fold_launch(const PgParams& p, bool f16_cache, uint32_t groups, uint32_t most, hipStream_t s);

// Heads of up to 256 dims by kernels for the next of these multiples of 32 (dims past a head are
// neither read nor written; their products are zeros).
#define PG_BY_DIM(hd, call)                          \
    do {                                             \
        const uint32_t nb_ = ((hd) + 31) / 32;       \
        if (nb_ <= 1) call(1);                       \
        else if (nb_ == 2) call(2);                  \
        else if (nb_ == 3) call(3);                  \
        else if (nb_ == 4) call(4);                  \
        else if (nb_ <= 6) call(6);                  \
        else call(8);                                \
    } while (0);

}  // namespace bchip
