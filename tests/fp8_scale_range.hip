/* nc_fp8.h's range of scales, on the host: rows stride blocks -> bytes. */
#include <cstdio>
#include <cstdlib>

#include "nc_fp8.h"

int main(int argc, char **argv) {
    if (argc != 4) return 2;
    printf("%lld\n", nc::f8_scale_range(atoll(argv[1]), atoll(argv[2]), atoi(argv[3])));
    return 0;
}
