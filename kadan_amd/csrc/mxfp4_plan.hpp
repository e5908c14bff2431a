// Which kernel of mxfp4_kernels.hpp a call runs, in which tile and how many K slices.  Plain host
// arithmetic over sizes and a number of compute units, so that tests can ask which variant a
// size reaches.
#pragma once
#include <algorithm>
#include <cmath>
#include <cstddef>

namespace kdq {
namespace mxfp4 {

constexpr size_t ceil_div(size_t a, size_t b) {
    return (a + b - 1) / b;
}

// What gemm_kernel multiplies: bf16 or MXFP4 rows of x by the packed form, or bf16 gradients by
// the transposed one (kOneTransposed, for plans only: a single matrix, where kTransposed has two).
enum Operands { kBf16, kFp4, kTransposed, kOneTransposed };

constexpr unsigned kTileFloats = 2 * 16 * 64;  // a wavefront's two result tiles
constexpr unsigned kStagedBytes = 32 * 1024;   // of x that decode_kernel passes through LDS

// Bytes between the rows of a staged x: 16 more than a row has, so that rows start in
// different banks.
constexpr unsigned staged_pitch(unsigned row_bytes) {
    return row_bytes + 16;
}

// How a product runs: `decode` (decode_kernel), or gemm_kernel with TT tiles of 32 rows of
// x, the groups splitting K or not, in `slices` of `part` chunks.
struct Plan {
    bool decode, split;
    int tt;
    unsigned tiles_n, tiles_m, slices, chunks, part;
    double cost;
};

// What a product in tiles of tt * 32 rows and `slices` K slices takes, in microseconds, up to
// what every choice shares: a workgroup's fixed part and its turns, alone on a compute unit or
// beside another, and the slices' sum.  Fitted to sweeps over tt and slices at 18 sizes per
// kind: 64 x 14336 -> 4096 16 us in 6 slices of 32 rows, 18 in 14 of 64, 23 in 14 of 128;
// 333 x 2880 -> 2880 gated 14 us in tiles of 32, 20 of 64, 25 of 128; 512 x 4096 -> 14336 51 us
// in tiles of 128, 53 of 64, 60 of 32; 512 x 4096 -> 4096 18 of 32, 26 of 64, 30 of 128.
struct Cost {
    double fixed, turn, turn_of_two;
};

inline Cost cost_of(int ops, int tt) {
    if (ops == kFp4)
        return {2.0 + 0.75 * tt, 0.05 + 0.55 * tt, 0.1 + 1.35 * tt};
    const double fixed = 2.5 + 0.9 * tt;
    return ops >= kTransposed ? Cost{fixed, tt == 1 ? 0.5 : 0.4 + 0.3 * tt, 0.7 + 0.6 * tt}
                              : Cost{fixed, 0.03 + 0.33 * tt, 0.05 + 0.66 * tt};
}

inline size_t partial_bytes(const Plan& p, size_t m) {
    return p.decode || p.slices == 1
               ? 0
               : size_t(p.slices) * p.tiles_n * 4 * ceil_div(m, 32) * kTileFloats * 4;
}

inline Plan plan_gemm(size_t m, size_t wave_groups, size_t chunks, int ops, size_t cus) {
    Plan best{};
    const auto consider = [&](int tt, bool split, size_t slices) {
        Plan p{};
        p.tt = tt;
        p.split = split;
        p.tiles_n = unsigned(ceil_div(wave_groups, 4));
        p.tiles_m = unsigned(ceil_div(m, size_t(tt) * (split ? 32 : 64)));
        p.chunks = unsigned(chunks);
        const unsigned sets = split && ops != kTransposed ? 2 : 1, unit = ops == kFp4 ? 1 : 4;
        p.part = unsigned(ceil_div(ceil_div(chunks, slices * sets), unit) * unit);
        p.slices = unsigned(ceil_div(chunks, size_t(p.part) * sets));
        const Cost c = cost_of(ops, tt);
        const bool shared = tt == 1 || (tt == 2 && ops != kFp4);
        const size_t tiles = size_t(p.tiles_n) * p.tiles_m;
        if (best.slices && tiles * 512 > UINT32_MAX)
            return;  // (a launch's threads are counted in 32 bits; the largest tiles come first)
        const size_t each = ceil_div(tiles * p.slices, cus);  // workgroups of a compute unit
        const double alone = c.fixed + p.part * c.turn, both = c.fixed + p.part * c.turn_of_two;
        // (two to a unit begin and end together: what their turns hide is paid once)
        double t = shared ? double(each / 2) * both + double(each % 2) * alone +
                                (each > 1 ? 1.5 : 0.0)
                          : double(each) * (split ? alone : 0.93 * alone);
        if (p.slices > 1)  // (the backward pass's third launch, which is its caller's time too)
            t += (ops >= kTransposed ? 4.5 : 3.5) + double(partial_bytes(p, m)) / 2.5e6;
        if (!best.slices || t < best.cost) {
            best = p;
            best.cost = t;
        }
    };
    for (int tt = 4; tt >= 1; --tt) {  // (slices up to two workgroups a compute unit)
        const size_t tiles = ceil_div(wave_groups, 4) * ceil_div(m, size_t(tt) * 32);
        const size_t most = std::min<size_t>({16, std::max<size_t>(1, 2 * cus / tiles),
                                              ceil_div(chunks, ops == kFp4 ? 2 : 4)});
        for (size_t slices = 1; slices <= most; ++slices)
            consider(tt, true, slices);
    }
    if (ops == kFp4)
        consider(4, false, 1);
    return best;
}

// How decode_kernel runs: whole blocks of 32 rows a workgroup (`wide`) where those fill the
// compute units, 16 rows of x or `tb` times as many, `waves` wavefronts of `units` units of 128
// values each, x through LDS (`staged`) or read by every wavefront.
struct DecodeShape {
    bool wide, staged;
    unsigned tb, waves, units;
};

// (1 row, 14336 -> 4096: 8.7 us over 16 wavefronts, 9.9 over 8; the gated projection's
// two matrices 14.9 and 14.1; 4096 -> 4096 5.5 and 4.9; 4096 -> 14336 13.1 and 8.1)
inline DecodeShape decode_shape(size_t m, size_t n, size_t k, bool gated, bool fp4, size_t cus) {
    DecodeShape s{};
    const size_t units = ceil_div(k, 128), row_bytes = fp4 ? k / 2 : k * 2;
    s.wide = ceil_div(n, 32) >= cus && m <= 32;
    s.tb = fp4 && m > 32 ? 4 : m > 16 ? 2 : 1;
    s.waves = units <= 8 ? 2 : units <= 16 ? 4 : units <= 48 || s.wide || gated || m > 32 ? 8 : 16;
    s.units = unsigned(ceil_div(ceil_div(units, s.waves), 2) * 2);
    s.staged = m <= 16 && m * staged_pitch(unsigned(row_bytes)) <= kStagedBytes &&
               m * row_bytes <= s.waves * 64 * 16 * 8;
    return s;
}

// What decode_kernel takes, in microseconds: its weights at 6 GB/ms, and each workgroup's own
// reading of x (m rows of row_bytes; none to speak of where x is staged, up to 16 rows) at what
// a compute unit takes of strided rows, 33 KB/us.  Swept against gemm_kernel over 11 sizes per
// kind and 1 to 64 rows: 4096 -> 14336 8 rows 10.7 us against 12.1, 16 rows 13.5 against 12.3;
// 14336 -> 4096 4 rows 11.2 against 12.6, 8 rows 14.0 against 12.7; 8192 -> 1024 12 rows 9.1
// against 9.3, 20 rows 14.6 against 9.4; 2880 -> 2880 20 rows 7.5 against 8.2, 32 rows 9.4
// against 8.3.  Rows of short K and wide outputs: 512 -> 131072 17 rows 17.4 against 10.1, 512 ->
// 4096 32 rows 3.6 against 4.5; MXFP4 896 -> 65536 64 rows 25.5 against 11.9, 17 rows 10.6
// against 10.3, 512 -> 262144 17 rows 20.6 against 25.7 (which the estimate misses: the GEMM's
// many rounds of short tiles are dearer than it counts).  What a workgroup costs by itself is in
// neither side: 128 -> 131072 1 row 10.5 against 7.1.
// Where x takes less than 2.5 us no plan of gemm_kernel is the quicker, and none is made: it
// would cost the caller about a microsecond.
struct DecodeCost {
    double weights, x;
    bool certain() const {
        return x < 2.5;
    }
    bool quicker_than(const Plan& gemm, bool fp4) const {
        return certain() || x + weights < gemm.cost - (fp4 ? 1.0 : 3.0);
    }
};

inline DecodeCost decode_cost(size_t m, size_t n, size_t k, bool gated, bool fp4, size_t cus) {
    const DecodeShape s = decode_shape(m, n, k, gated, fp4, cus);
    const double rounds = std::max(1.0, double(ceil_div(n, s.wide ? 32 : 16)) / double(cus));
    const size_t row_bytes = fp4 ? k / 2 : k * 2, weight_bytes = n * k * 17 / 32 * (gated ? 2 : 1);
    return {double(weight_bytes) / 6.0e6,
            s.staged ? 0.0 : double(m * row_bytes) * rounds / 33.0e3};
}

inline Plan decode_plan() {
    Plan p{};
    p.decode = true;
    return p;
}

inline Plan plan_product(size_t m, size_t n, size_t k, bool fp4, size_t cus) {
    const bool few = m <= (fp4 ? 64 : 32);
    const DecodeCost d = few ? decode_cost(m, n, k, false, fp4, cus) : DecodeCost{};
    if (few && d.certain())
        return decode_plan();
    const Plan p = plan_gemm(m, ceil_div(n, 64), ceil_div(k, fp4 ? 256 : 64), fp4 ? kFp4 : kBf16,
                             cus);
    return few && d.quicker_than(p, fp4) ? decode_plan() : p;
}

inline Plan plan_gated(size_t m, size_t n, size_t k, bool kept, size_t cus) {
    const bool few = !kept && m <= 32;
    const DecodeCost d = few ? decode_cost(m, n, k, true, false, cus) : DecodeCost{};
    if (few && d.certain())
        return decode_plan();
    const Plan p = plan_gemm(m, ceil_div(n, 32), ceil_div(k, 64), kBf16, cus);
    return few && d.quicker_than(p, false) ? decode_plan() : p;
}

// (decode_t_kernel is bound by decoding the weights, which half the compute units do where
// there are 4096 columns: 1 row of 14336 -> 4096 26 us against 21, of 2880 -> 2880 10.3
// against 13.0, 16 rows of that 15.0 against 13.2, 1 row of 1024 -> 8192 6.6 against 11.6)
inline Plan plan_backward(size_t m, size_t n, size_t k, size_t cus) {
    Plan p = plan_gemm(m, ceil_div(k, 64), ceil_div(n, 64), kTransposed, cus);
    const double units = double(ceil_div(n, 128)) * double(ceil_div(k / 32, cus));
    p.decode = m <= 32 && 2.5 + 0.2 * units * (1.0 + double(m) / 14) < p.cost;
    return p;
}

inline Plan plan_one_backward(size_t m, size_t n, size_t k, size_t cus) {
    return plan_gemm(m, ceil_div(k, 64), ceil_div(n, 64), kOneTransposed, cus);
}

// The most tiles of `rows` rows that m rows of x, sorted by expert, may make: an expert's last one
// may hold a single row.
constexpr size_t most_tiles(size_t m, size_t experts, size_t rows) {
    return (m + (rows - 1) * std::min(experts, m)) / rows;
}

// Tiles of `rows` rows that an expert's `count` rows make: in the low half of a word, and in the
// high half whether the last has at most half the rows (where `halves` tells such apart: it is then
// not in the low half).
constexpr unsigned tiles_of(unsigned count, unsigned rows, bool halves) {
    const unsigned tiles = (count + (halves ? rows / 2 - 1 : rows - 1)) / rows;
    return halves && count > tiles * rows ? tiles | 1u << 16 : tiles;
}

// What workgroup `block` of the experts' launch of gemm_kernel takes: a workgroup's share of whole
// tile `tile / tiles_n` (or half), or nothing. Workgroups go round the eight XCDs, and an XCD has
// its share of whole tiles, then of halves, all K slices of either before its workgroups of
// neither.
struct ExpertsItem {
    unsigned tile, slice;
    bool half, there;
};

constexpr ExpertsItem experts_item(unsigned block, unsigned whole, unsigned halves,
                                   unsigned tiles_n, unsigned slices) {
    const unsigned xcd = block % 8;
    unsigned turn = block / 8, tiles = whole * tiles_n * slices;
    unsigned share = tiles / 8 + (xcd < tiles % 8);
    const bool half = turn >= share;
    if (half) {
        turn -= share;
        tiles = halves * tiles_n * slices;
        share = tiles / 8 + (xcd < tiles % 8);
    }
    ExpertsItem item{xcd * (tiles / 8) + (xcd < tiles % 8 ? xcd : tiles % 8) + turn, 0, half,
                     turn < share};
    if (slices > 1) [[unlikely]] {
        const unsigned each = tiles / slices;
        item.slice = item.tile / (each ? each : 1);
        item.tile -= item.slice * each;
    }
    return item;
}

// Where a K slice's partial sums of row tile T (of 32 rows) of the launch's tile `spot` lie, for
// the wavefronts of row group G: in tiles of kTileFloats, of which there are partial_bytes' for
// `most` tiles of `tt` row tiles.
constexpr size_t partial_tile(unsigned slice, unsigned G, unsigned spot, unsigned T,
                              unsigned tiles_n, unsigned tt, unsigned most) {
    return (size_t(slice) * (tiles_n * 4) + G) * (most * tt) + spot * tt + T;
}

// Offsets that decrease may make more tiles than `most`: those have no partial sums.
constexpr bool has_partials(unsigned spot, unsigned most) {
    return spot < most;
}

// How the experts' products run: decode_kernel over tiles of 16 rows, or gemm_kernel over tiles of
// tt * 32; `most` tiles at most (the device alone knows how many), each in tiles_n workgroups.
//
// gemm_kernel takes weights at the memory's rate as soon as there are workgroups of it for most
// compute units, also where an expert has one row (256 sorted rows over 25 of 32 experts of
// 2880 x 2880, gated: 41 us, 235 MB at 5.7 TB/s; decode_kernel 50).  Fewer, as for a token or two,
// leave units without any, and decode_kernel's narrower shares are the quicker: 1 token to 4 of 32
// experts gated 10.7 us against 15.5, then down 7.7 against 12.8; 2 tokens gated (184 workgroups)
// 15.9 against 14.4, down (96) 9.8 against 12.8.  It reads a row of x once for each of its
// workgroups: 16 tokens to 2 of 8 experts 5632 -> 4096 20.5 us against 20.4, 32 tokens 28 against
// 21.
//
// Tiles of 64 rows (two workgroups of either share a compute unit; a half that is empty is not
// multiplied) decode a weight once for twice the rows, tiles of 32 are more, and fill the last
// round of workgroups better.  Rows an expert, in us over tiles of 32 and of 64: 32 experts of 2880
// x 2880 gated 16 59, 57; 32 70, 73; 64 100, 91; down 16 33, 37; 32 40, 39; 64 52, 56; 128 83, 80;
// their gradients gated 16 76, 83; 32 100, 89; down 16 32, 38; 32 49, 42; 64 65, 62; 128 experts of
// 2048 x 768 gated 32 53, 52; 64 73, 67; down (K of 768, where a workgroup's fixed part is the
// larger) 32 38, 38; 64 54, 50; gradients gated 16 55, 54; 32 71, 67; down 16 24, 27; 32 34, 29.
// (That border of K, 1536, lies between the two widths measured, 768 and 2880.)
// Tiles of 96 and 128 rows have a unit to themselves and lose by 5 to 50 % up to 512 rows an
// expert; at 2048 they are within 2 % of those of 64.
struct ExpertsPlan {
    bool decode;
    DecodeShape shape;
    int tt;
    size_t tiles_n, most;
    unsigned slices, chunks, part;  // of K, in chunks
};

inline size_t partial_bytes(const ExpertsPlan& p) {
    return p.decode || p.slices == 1
               ? 0
               : size_t(p.slices) * p.tiles_n * 4 * p.most * p.tt * kTileFloats * 4;
}

// K slices where the tiles are too few to fill the compute units: by plan_gemm's estimate, and no
// shorter than `reached` experts' `bytes` take, longer where few workgroups ask for them; over the
// tiles that as many experts with half a tile more than whole ones would make. `sets`: parts of K
// that a workgroup takes, of `unit` chunks.
// (measured calls, us by slices, the gated backward's with its gate gradients:
//  gated backward of 4 rows, 3392 -> 1024: 36.6 as one, 16.8 in 6, 15.7 in 8, 16.2 in 16
//  594 rows of 6 experts, 5920 -> 416: 88 as one, 31.7 in 6, 29.7 in 8, 33.0 in 12; product 37.6,
//  19.5 in 6, 23.5 in 12
//  64 rows of 8 experts, 5632 -> 4096: backward 60 as one, 44 in 2, 48 in 4; product, which reads
//  92 MB, 24.7, 22.8, 26.2)
inline void slice_experts(ExpertsPlan& p, size_t m, size_t reached, double bytes, size_t chunks,
                          size_t sets, size_t unit, int ops, size_t cus) {
    const double tiles =
        std::min(double(p.most), std::max(double(m) / double(p.tt * 32) + 0.5 * double(reached),
                                          0.85 * double(reached)));
    const Cost c = cost_of(ops, p.tt);
    double best = 0;
    p.chunks = unsigned(chunks);
    for (size_t slices = 1; slices <= 16; ++slices) {
        const size_t part = ceil_div(ceil_div(chunks, slices * sets), unit) * unit;
        const size_t real = ceil_div(chunks, part * sets);
        const double groups = tiles * double(p.tiles_n) * double(real);
        const double each = std::ceil(groups / double(cus));
        const double alone = c.fixed + double(part) * c.turn;
        const double both = c.fixed + double(part) * c.turn_of_two;
        const double rate = 4.5e6 * std::sqrt(std::min(1.0, groups / (0.75 * double(cus))));
        double t = std::max(each <= 1 ? alone : each / 2 * both, bytes / rate);
        if (real > 1)
            t += 2 + 0.25 * double(real) + groups * p.tt * 4 * kTileFloats * 4 / 2e6;
        if (slices == 1 || t < best) {
            best = slices == 1 ? 0.9 * t : t;  // (a tenth less, or not at all)
            p.slices = unsigned(real);
            p.part = unsigned(part);
        }
    }
}

inline ExpertsPlan plan_experts(size_t m, size_t experts, size_t n, size_t k, bool gated,
                                bool kept, size_t cus) {
    ExpertsPlan p{};
    const size_t reached = std::min(experts, m), mean = m / reached;  // (at most, at least)
    p.tiles_n = ceil_div(n, gated ? 128 : 256);
    p.decode = !(gated && kept) && p.tiles_n * reached * 9 <= cus * 5 && mean <= 4;
    if (p.decode) {
        // (runs of four units, a batch whose loads are all in flight at once, and where two matrices
        // are twice as many, of eight: gated 2880 -> 2880 of a token 10.7 us over 3 wavefronts, 11.4
        // over 4, 12.1 over 6, 2048 -> 768 6.2 over 4, 7.3 over 2; down 5632 -> 4096 8.2 over 11,
        // 9.3 over 6; the border, 2048, is the last width measured the one way, 2880 the next)
        const size_t units = ceil_div(k, 128), run = gated && units > 16 ? 8 : 4;
        p.shape.waves = unsigned(std::min<size_t>(ceil_div(units, run), 16));
        p.shape.units = unsigned(ceil_div(ceil_div(units, p.shape.waves), 2) * 2);
        // (whole blocks of 32 rows where there is work enough for half as many workgroups, each
        // counted as a wavefront more than it has: down 2880 -> 2880 of a token 7.9 us against 7.7,
        // of two 9.8 against 10.9; 5632 -> 4096 of a token 8.1 against 8.7)
        p.shape.wide = !gated && ceil_div(n, 16) * reached * (p.shape.waves + 1) >= 21 * cus;
        p.shape.tb = 1;
        p.most = most_tiles(m, experts, 16);
        return p;
    }
    p.tt = mean < (gated || k <= 1536 ? 48 : 96) ? 1 : 2;
    p.most = most_tiles(m, experts, size_t(p.tt) * 32);
    slice_experts(p, m, reached, double(reached) * double(n * k) * (gated ? 17 : 8.5) / 16,
                  ceil_div(k, 64), 2, gated ? 4 : 2, kBf16, cus);
    return p;
}

// (`gated`: two matrices, each of a wavefront group's own)
inline ExpertsPlan plan_experts_backward(size_t m, size_t experts, size_t n, size_t k, bool gated,
                                         size_t cus) {
    ExpertsPlan p{};
    const size_t reached = std::min(experts, m);
    p.tt = m / reached < 24 ? 1 : 2;
    p.tiles_n = ceil_div(k, 256);
    p.most = most_tiles(m, experts, size_t(p.tt) * 32);
    slice_experts(p, m, reached, double(reached) * double(n * k) * (gated ? 17 : 8.5) / 16,
                  ceil_div(n, 64), gated ? 1 : 2, 4, kTransposed, cus);
    return p;
}

}  // namespace mxfp4
}  // namespace kdq
