// An expert's rows from two offsets (mx_grouped_gemm.cuh), whatever the offsets are: inside the matrix, in order.
#include <cstdio>
#include <cstdlib>

#include "../../catccos_b200/csrc/mx_grouped_gemm.cuh"

int main()
{
    const int32_t values[] = {INT32_MIN, -5, -1, 0, 1, 39, 40, 41, INT32_MAX};
    for (uint32_t rows : {1u, 40u, 0x7FFFFFFFu}) {
        for (int32_t lo : values) {
            for (int32_t hi : values) {
                uint32_t begin, end;
                catccos::grouped_rows(lo, hi, rows, begin, end);
                const bool good = lo >= 0 && hi >= lo && (uint32_t)hi <= rows;
                if (begin > end || end > rows || (good && (begin != (uint32_t)lo || end != (uint32_t)hi)) || (hi <= lo && begin != end)) {
                    printf("rows %u offsets %d %d: [%u, %u)\n", rows, lo, hi, begin, end);
                    return 1;
                }
            }
        }
    }
    printf("grouped rows ok\n");
    return 0;
}
