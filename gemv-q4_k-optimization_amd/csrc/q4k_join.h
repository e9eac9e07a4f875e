// q4k_join.h -- who does what in a workgroup of 256 threads that joins the partial
// results of attention rows: head_dim / 4 threads, four dimensions each, are a group;
// `groups` of them take the parts of one row by turns and meet in LDS.
// Plain C++, for the kernels, the host's plan and tests alike.
#pragma once

namespace q4k {

constexpr int kJoinThreads = 256;

// Groups of a row and rows of a workgroup: groups for the parts of a row, so that each reads its up
// to four at once.
struct JoinSplit {
    int groups, rows;
};
constexpr JoinSplit join_split(int head_dim, long long parts) {
    const int all = kJoinThreads / (head_dim / 4);
    int groups = 1;
    while (groups * 2 <= all && groups * 4 < parts) groups *= 2;
    return JoinSplit{groups, all / groups};
}

struct JoinThread {
    int d4, sub, which;  // four dimensions, group of the row, row of the workgroup
    bool there;          // groups that are left over, and threads of no whole group, have no row
    constexpr JoinThread(int thread, int head_dim, int groups, int rows)
        : d4(thread % (head_dim / 4)), sub(thread / (head_dim / 4) % groups), which(thread / (head_dim / 4) / groups), there(which < rows) {}
    // It adds up what the row's groups left in LDS, and writes the row.
    constexpr bool collects() const { return there && sub == 0; }
    // Where in LDS the row's group `i` left its sum of these dimensions.
    static constexpr int place(int thread, int head_dim, int i) { return thread + i * (head_dim / 4); }
};

}  // namespace q4k
