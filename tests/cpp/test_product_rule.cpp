// The kernel that the products choose for calls read from stdin: kind grouped n_rows n_groups rows k_bytes a line.
#include "vbm_product_rule.hpp"

#include <cstdio>

using namespace vbm;

int main() {
    const char * names[] = {"few8", "few16", "stream8_4", "stream8_8", "stream16_4", "stream16_8", "tile256x256", "tile256x160", "tile256x128",
                            "tile128x64", "tile64x32"};
    int kind, grouped;
    long long n_rows, n_groups, rows, k_bytes;
    while (std::scanf("%d %d %lld %lld %lld %lld", &kind, &grouped, &n_rows, &n_groups, &rows, &k_bytes) == 6) {
        const ProductSize s{grouped != 0, n_rows, n_groups, rows, (k_bytes + 127) / 128};
        ProductKernel k{};
        switch (kind) {
            case kF8Wide: k = product_kernel<kF8Wide>(s); break;
            case kF8: k = product_kernel<kF8>(s); break;
            case kF16: k = product_kernel<kF16>(s); break;
            default: k = product_kernel<kBF16>(s);
        }
        std::printf("%s\n", names[static_cast<int>(k)]);
    }
    return 0;
}
