// Prints what kadan_amd/csrc/mxfp4_plan.hpp picks for the calls on standard input, one a line:
//   linear m n k | back m n k | experts m experts n k gated kept |
//   experts_back m experts n k gated | tiles m experts rows
// as "decode wide staged tb", "gemm tt split sliced", "experts decode wide", "experts gemm tt sliced" or
// a number of tiles, on `argv[1]` compute units.
#include "mxfp4_plan.hpp"

#include <cstdlib>
#include <iostream>
#include <string>

using namespace kdq::mxfp4;

int main(int, char** argv) {
    const size_t cus = std::strtoul(argv[1], nullptr, 10);
    std::string path;
    while (std::cin >> path) {
        size_t m, a, b, c = 0, gated = 0, kept = 0;
        std::cin >> m >> a >> b;
        if (path == "tiles") {
            std::cout << most_tiles(m, a, b) << '\n';
            continue;
        }
        if (path == "linear" || path == "back") {
            const Plan p = path == "linear" ? plan_product(m, a, b, false, cus)
                                            : plan_one_backward(m, a, b, cus);
            if (p.decode) {
                const DecodeShape s = decode_shape(m, a, b, false, false, cus);
                std::cout << "decode " << s.wide << ' ' << s.staged << ' ' << s.tb << '\n';
            } else {
                std::cout << "gemm " << p.tt << ' ' << p.split << ' ' << (p.slices > 1) << '\n';
            }
            continue;
        }
        std::cin >> c >> gated;
        if (path == "experts")
            std::cin >> kept;
        const ExpertsPlan p = path == "experts" ? plan_experts(m, a, b, c, gated, kept, cus)
                                                : plan_experts_backward(m, a, b, c, gated, cus);
        if (p.decode)
            std::cout << "experts decode " << p.shape.wide << '\n';
        else
            std::cout << "experts gemm " << p.tt << ' ' << (p.slices > 1) << '\n';
    }
}
