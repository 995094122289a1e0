/*
 * mzs_policy_plan.h — how a call on policy rows becomes launches: host arithmetic alone, so that mzs_policy_workspace, the launches
 * and a test without a GPU read the same plan.
 */
#ifndef MZS_POLICY_PLAN_H
#define MZS_POLICY_PLAN_H

#include <cstddef>
#include <cstdint>

#include "../../include/mzsearch.h"

namespace mzs {

constexpr int kPolicyBlock = 256;    /* threads that walk a chunk of a wide row                     */
constexpr int kPolicyAhead = 4;      /* 16-byte vectors a thread of them has in flight              */
constexpr int kPolicyStripLanes = 4; /* neighbouring threads whose vectors make a strip             */
constexpr int kPolicyStrips = kPolicyBlock / kPolicyStripLanes; /* strips of a chunk               */
constexpr int kPolicyWaveVecs = 16;  /* most vectors a lane of a wave holds of a row                */
constexpr int kPolicyLanesMost = 8;  /* widest row that one lane has, a logit at a time             */

/* rows in a wave's registers */
inline bool policy_fits_wave(int64_t n, int per) { return n >= per && n <= (int64_t)64 * kPolicyWaveVecs * per; }

/* How a wide row is cut: `chunks` blocks a row, each thread `vecs` vectors of `per` logits.  Only few and long rows are: a block alone
 * reads 12000 bf16 a us, and the join costs a launch and a second search (us whole / cut, without alternatives and with five, logits from
 * memory: 8 x 100000 bf16 - and 15 / 10, 64 of them 13 / 11 and 17 / 15, 100 13 / 13, 160 16 / 19 and 20 / 23; 8 x 50000 - and 10 / 10; 8 x 20000 -
 * and 7.7 / 9.7, 64 5.5 / 6.9 and 8.4 / 11; fp32 32 x 100000 19 / 18 with, one of 30000 8 / 9). */
struct PolicyCut {
    int chunks, vecs;
};
constexpr int64_t kPolicyCutLeast = 49152;
inline PolicyCut policy_cut(int64_t rows, int64_t n, int per) {
    const int64_t each = (int64_t)kPolicyBlock * per, all = (n + each - 1) / each; /* vectors a thread would have of a whole row */
    int64_t chunks = 1;
    if (rows < MZS_POLICY_MANY && n >= kPolicyCutLeast) chunks = (8192 + rows - 1) / rows;
    if (chunks > kPolicyBlock) chunks = kPolicyBlock;
    if (chunks > all) chunks = all;
    PolicyCut c;
    c.vecs = (int)((all + chunks - 1) / chunks);
    if (chunks > 1 && c.vecs > kPolicyAhead) c.vecs = (c.vecs + kPolicyAhead - 1) / kPolicyAhead * kPolicyAhead; /* whole groups */
    c.chunks = (int)((all + c.vecs - 1) / c.vecs);
    return c;
}

/* The plan of a call of rows >= 1: made once, from the call's own rows, whatever number of them a launch takes. */
struct PolicyPlan {
    PolicyCut cut;    /* of every row that blocks walk, in every launch */
    int64_t slab;     /* rows of a launch                                */
    size_t workspace; /* bytes                                           */
};
inline size_t policy_launch_bytes(const PolicyCut& c, int64_t rows, int top) { /* what a launch of so many cut rows writes there */
    return c.chunks == 1 ? 0 : sizeof(float) * (size_t)rows * c.chunks * (3 + (top > 0 ? kPolicyStrips : 0));
}
inline PolicyPlan policy_plan(int64_t rows, int64_t n, int per, int top) {
    PolicyPlan p;
    p.cut = policy_cut(rows, n, per);
    /* blocks times threads stay below 2^32: a wave a row at most, or a block, which a row that a wave could hold gets for its
     * alternatives and its gradient */
    p.slab = n <= MZS_POLICY_NARROW ? (int64_t)1 << 24 : (int64_t)1 << 20;
    p.workspace = policy_launch_bytes(p.cut, rows, top);
    return p;
}
/* calls launch(first row, rows, plan) for each launch, in order */
template <typename F>
inline void policy_launches(int64_t rows, const PolicyPlan& plan, F launch) {
    for (int64_t r = 0; r < rows; r += plan.slab) launch(r, rows - r < plan.slab ? rows - r : plan.slab, plan);
}

}  // namespace mzs
#endif
