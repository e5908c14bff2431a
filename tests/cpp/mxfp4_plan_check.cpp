// Prints what kadan_amd/csrc/mxfp4_plan.hpp picks for the calls on standard input, one a line:
//   product m n k quantized | gated m n k kept | backward m n k
// as "decode wide staged tb waves" or "gemm tt split slices", on `argv[1]` compute units.
#include "mxfp4_plan.hpp"

#include <cstdlib>
#include <iostream>
#include <string>

using namespace kdq::mxfp4;

int main(int, char** argv) {
    const size_t cus = std::strtoul(argv[1], nullptr, 10);
    std::string path;
    size_t m, n, k, flag;
    while (std::cin >> path >> m >> n >> k) {
        flag = 0;
        if (path != "backward")
            std::cin >> flag;
        const Plan p = path == "product" ? plan_product(m, n, k, flag != 0, cus)
                       : path == "gated" ? plan_gated(m, n, k, flag != 0, cus)
                                         : plan_backward(m, n, k, cus);
        if (!p.decode) {
            std::cout << "gemm " << p.tt << ' ' << p.split << ' ' << p.slices << '\n';
        } else if (path == "backward") {
            std::cout << "decode 0 0 " << (m <= 16 ? 1 : 2) << " 0\n";
        } else {
            const bool gated = path == "gated";
            const DecodeShape s = decode_shape(m, n, k, gated, !gated && flag, cus);
            std::cout << "decode " << s.wide << ' ' << s.staged << ' ' << s.tb << ' ' << s.waves
                      << '\n';
        }
    }
}
