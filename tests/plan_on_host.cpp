// The plan of attention over pages (csrc/paged_plan.cuh, copied beside this file), laid by a block of any number of threads on the host.
#include "host_block.h"
#include "paged_plan.cuh"

// out: blocks of the second way, units of a worker and of the line for each way, then 4 * (sets + 1) places and n_req + 1 rows that share a prefix; 0 if the lengths are refused
extern "C" int plan_on_host(const b200_paged_attn_args *a, int few_most, int big, int blocks, int few_warps, int ratio, int threads, int *out)
{
    const int G = a->n_q / a->n_kv, sets = a->n_req + a->n_groups;
    Shape shape = {};
    shape.by_g = div_of(G); shape.by_kv = div_of(a->n_kv);
    shape.few_most = few_most; shape.big = big; shape.blocks = blocks; shape.few_warps = few_warps; shape.ratio = ratio;
    shape.each = (sets + threads - 1) / threads;
    shape.row_step[0] = (Cut<0>::ROWS * 256 + G - 1) / G; shape.row_step[1] = (Cut<1>::ROWS * 256 + G - 1) / G;
    std::vector<char> mem(plan_bytes(a->n_req, a->n_groups));
    Plan plan = {};
    bool fine = false;
    blockIdx.x = 0;
    host_block::run(threads, [&] { const bool ok = make_plan(*a, shape, mem.data(), plan); if (threadIdx.x == 0) fine = ok; });
    if (!fine) return 0;
    const int head[5] = {plan.many_blocks, plan.per[0], plan.per[1], plan.units[0], plan.units[1]};
    memcpy(out, head, sizeof head);
    memcpy(out + 5, mem.data(), 4 * (sets + 1) * sizeof(int));
    memcpy(out + 5 + 4 * (sets + 1), plan.small, (a->n_req + 1) * sizeof(int));
    return 1;
}
