// Reads calls (B P H_q H_kv d kv_dtype max_keys window asked), one a line, and
// prints each one's form and splits: rows, groups of waves, splits.
#include <cstdio>

#include "paged_plan.h"

int main() {
    int a[9];
    while (scanf("%d %d %d %d %d %d %d %d %d", a, a + 1, a + 2, a + 3, a + 4, a + 5, a + 6, a + 7, a + 8) == 9) {
        const ie::PagedPlan p = ie::paged_plan(a[0], a[1], a[2], a[3], a[4], a[5], a[6], a[7], a[8]);
        printf("%d %d %d\n", p.rows, p.groups, p.splits);
    }
}
