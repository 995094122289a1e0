/* Plans of policy-row calls (muzero_amd/csrc/mzs_policy_plan.h) over rows and logits from argv: "rows logits logits-per-vector top" each.
 * Prints the workspace of each; fails if its launches do not add up to the call or need more than the workspace together or alone. */
#include <cstdio>
#include <cstdlib>

#include "../../muzero_amd/csrc/mzs_policy_plan.h"

int main(int argc, char** argv) {
    int bad = 0;
    for (int i = 1; i + 3 < argc; i += 4) {
        const int64_t rows = std::atoll(argv[i]), n = std::atoll(argv[i + 1]);
        const int per = std::atoi(argv[i + 2]), top = std::atoi(argv[i + 3]);
        const mzs::PolicyPlan call = mzs::policy_plan(rows, n, per, top);
        int64_t next = 0, launches = 0;
        mzs::policy_launches(rows, call, [&](int64_t first, int64_t count, const mzs::PolicyPlan& plan) {
            const mzs::PolicyCut c = plan.cut;
            const int64_t chunk = (int64_t)c.vecs * mzs::kPolicyBlock * per;
            bad += first != next || count < 1;
            bad += mzs::policy_launch_bytes(c, count, top) > call.workspace;        /* what the launch writes */
            bad += c.chunks != call.cut.chunks || c.vecs != call.cut.vecs;
            bad += c.chunks < 1 || c.chunks > mzs::kPolicyBlock;                    /* a thread of the join each */
            bad += (c.chunks * chunk < n || (c.chunks - 1) * chunk >= n);   /* the chunks are the row, none is empty */
            bad += n > MZS_POLICY_NARROW && count * c.chunks * mzs::kPolicyBlock >= (int64_t)1 << 32; /* a block a row */
            next = first + count, ++launches;
        });
        bad += next != rows;
        bad += (n <= MZS_POLICY_NARROW || rows >= MZS_POLICY_MANY) && call.workspace > 0; /* the header's promise */
        std::printf("%lld %zu %d\n", (long long)launches, call.workspace, call.cut.chunks);
    }
    std::printf("bad %d\n", bad);
    return bad != 0;
}
