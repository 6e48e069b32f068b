// Reads calls (rows experts n k grouped pairs_only block_rows split_k cta_pair num_sms), prints the plan of each (rows parts).
#include <cstdio>

#include "../../catccos_b200/csrc/block_plan.hpp"

int main()
{
    using namespace catccos;
    BlockCall c;
    BlockChoice o;
    unsigned grouped, pairs_only, num_sms;
    while (scanf("%u %u %u %u %u %u %d %d %d %u", &c.rows, &c.experts, &c.n, &c.k, &grouped, &pairs_only, &o.block_rows, &o.split_k, &o.cta_pair, &num_sms) == 10) {
        c.grouped = grouped != 0;
        c.pairs_only = pairs_only != 0;
        const BlockPlan p = plan_block_gemm(c, o, num_sms);
        printf("%u %u\n", p.rows, p.parts);
    }
}
