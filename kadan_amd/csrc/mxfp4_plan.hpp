// Which kernel of mxfp4_dense.hip a call runs, in which tile and how many K slices.  Plain host
// arithmetic over sizes and a number of compute units, so that tests can ask which variant a
// size reaches.
#pragma once
#include <algorithm>
#include <cstddef>

namespace kdq {
namespace mxfp4 {

constexpr size_t ceil_div(size_t a, size_t b) {
    return (a + b - 1) / b;
}

// What gemm_kernel multiplies: bf16 or MXFP4 rows of x by the packed form, or bf16 gradients by
// the transposed one.
enum Operands { kBf16, kFp4, kTransposed };

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
    return ops == kTransposed ? Cost{fixed, tt == 1 ? 0.5 : 0.4 + 0.3 * tt, 0.7 + 0.6 * tt}
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
            t += (ops == kTransposed ? 4.5 : 3.5) + double(partial_bytes(p, m)) / 2.5e6;
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

}  // namespace mxfp4
}  // namespace kdq
