// Device-side reading of a paged step's lengths, shared by the paged-cache
// kernels.
#pragma once

#include "../../include/affon_b200.h"
#include "common.cuh"
#include "internal.h"

namespace afb {

// Rows [first, last) and cached length of one sequence; ok says that they fit
// the step's buffers and the page table.
struct SeqSpan {
    int first, last, ctx;
    bool ok;
};
AFB_DEVICE SeqSpan seq_span(const PagedShape &s, const PagedStep &t, int seq) {
    SeqSpan r;
    r.first = t.cu_nodes[seq];
    r.last = t.cu_nodes[seq + 1];
    r.ctx = t.ctx_lens[seq];
    const int64_t n = static_cast<int64_t>(r.last) - r.first;
    r.ok = r.first >= 0 && n >= 0 && n <= s.max_nodes && r.last <= s.rows && r.ctx >= 0 &&
           r.ctx + n <= (s.ld_table << s.page_shift);
    return r;
}

}  // namespace afb
