// What the workgroups of an experts' launch of gemm_kernel do with the offsets on standard input,
// by the arithmetic of kadan_amd/csrc/mxfp4_plan.hpp that the kernel uses.  A line:
//   linear|gated|back|gated_back m experts n k offset ..   (experts + 1 offsets)
// Prints the launch's K slices, the tiles of partial sums that there are, how many of them are
// reached at most, the tiles (of x rows, matrix rows and K slices) that the offsets ask for, and
// how many of those no workgroup or more than one takes; "decode" where decode_kernel runs.
// argv[1]: compute units.
#include "mxfp4_plan.hpp"

#include <algorithm>
#include <cstdlib>
#include <iostream>
#include <map>
#include <string>
#include <tuple>
#include <vector>

using namespace kdq::mxfp4;

namespace {
// Expert, first row: the tile that number `t` among the whole tiles (or halves) is, and the
// tiles and the number of the expert's first.
struct Place {
    unsigned expert, first, end, before, tiles;
};

Place of(const std::vector<long>& at, unsigned rows, bool halves, unsigned t, bool half) {
    unsigned before = 0;
    for (unsigned e = 0; e + 1 < at.size(); ++e) {
        const unsigned first = unsigned(at[e]), end = unsigned(std::max(at[e], at[e + 1]));
        const unsigned tiles = tiles_of(end - first, rows, halves);
        const unsigned count = half ? tiles >> 16 : tiles & 0xffff;
        if (t >= before && t < before + count)
            return {e, first + (half ? (tiles & 0xffff) * rows : 0), end, before, count};
        before += count;
    }
    return {};
}
}  // namespace

int main(int, char** argv) {
    const size_t cus = std::strtoul(argv[1], nullptr, 10);
    std::string path;
    while (std::cin >> path) {
        size_t m, experts, n, k;
        std::cin >> m >> experts >> n >> k;
        std::vector<long> at(experts + 1);
        for (long& v : at) {
            std::cin >> v;
            v = std::clamp(v, 0l, long(m));
        }
        const bool gated = path[0] == 'g', back = path.ends_with("back");
        const ExpertsPlan p = back ? plan_experts_backward(m, experts, n, k, gated, cus)
                                   : plan_experts(m, experts, n, k, gated, gated, cus);
        if (p.decode) {
            std::cout << "decode\n";
            continue;
        }
        const unsigned rows = unsigned(p.tt) * 32, tiles_n = unsigned(p.tiles_n);
        const unsigned most = unsigned(p.most), tt = unsigned(p.tt);
        unsigned whole = 0, halves = 0;
        for (size_t e = 0; e < experts; ++e) {
            const unsigned tiles =
                tiles_of(unsigned(std::max(at[e], at[e + 1]) - at[e]), rows, tt > 1);
            whole += tiles & 0xffff, halves += tiles >> 16;
        }
        // (expert, row, matrix tile, slice): workgroups
        std::map<std::tuple<unsigned, unsigned, unsigned, unsigned>, int> taken;
        size_t reached = 0;
        const unsigned blocks = tiles_n * most * p.slices + 16;
        for (unsigned block = 0; block < blocks; ++block) {
            const ExpertsItem item = experts_item(block, whole, halves, tiles_n, p.slices);
            const Place q = of(at, rows, tt > 1, item.tile / tiles_n, item.half);
            if (!item.there || !q.tiles)
                continue;
            const unsigned within = item.tile - q.before * tiles_n;
            const unsigned first = q.first + within % q.tiles * rows;
            const unsigned spot = (item.half ? whole : 0) + q.before + within % q.tiles;
            if (p.slices > 1 && !has_partials(spot, most))
                continue;
            if (first >= q.end || within / q.tiles >= tiles_n || item.slice >= p.slices) {
                std::cout << "a workgroup past its expert\n";
                return 1;
            }
            ++taken[{q.expert, first, within / q.tiles, item.slice}];
            const unsigned row_tiles = (std::min(q.end - first, rows) + 31) / 32;
            if (p.slices > 1)
                reached = std::max(
                    reached, partial_tile(item.slice, within / q.tiles * 4 + 3, spot,
                                          row_tiles - 1, tiles_n, tt, most) + 1);
        }
        size_t asked = 0, wrong = 0;
        for (size_t e = 0; e < experts; ++e)
            for (unsigned row = unsigned(at[e]); long(row) < at[e + 1]; row += rows)
                for (unsigned tile = 0; tile < tiles_n; ++tile)
                    for (unsigned slice = 0; slice < p.slices; ++slice, ++asked) {
                        const auto found = taken.find({unsigned(e), row, tile, slice});
                        wrong += found == taken.end() || found->second != 1;
                    }
        std::cout << p.slices << ' ' << partial_bytes(p) / (kTileFloats * 4) << ' ' << reached
                  << ' ' << asked << ' ' << wrong << '\n';
    }
}
