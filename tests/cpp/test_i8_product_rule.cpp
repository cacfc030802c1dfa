// The kernel that the integer products choose for calls read from stdin: grouped n_rows n_groups rows k a line.
#include "vbm_product_rule.hpp"

#include <cstdio>

using namespace vbm;

int main() {
    const char * names[] = {"few8", "few16", "stream8_4", "stream8_8", "stream16_4", "stream16_8", "tile256x256", "tile256x160", "tile256x128",
                            "tile128x64", "tile64x32"};
    int grouped;
    long long n_rows, n_groups, rows, k;
    while (std::scanf("%d %lld %lld %lld %lld", &grouped, &n_rows, &n_groups, &rows, &k) == 5)
        std::printf("%s\n", names[static_cast<int>(product_kernel<kI8>(ProductSize{grouped != 0, n_rows, n_groups, rows, (k + 127) / 128}))]);
    return 0;
}
