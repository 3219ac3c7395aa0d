// Validation of a batch's lengths and page table (host_plan.cpp), shared by ggr_batch_check and ggr_batch_set.
#pragma once

#include <cstdint>

namespace ggr {

struct BatchTotals {
    int64_t tokens, rows, entries;  // new tokens, cached tokens, page table entries in use
};

// GGR_OK and the totals, or a status and what is wrong. page_size 0: packed prompts.
int batch_check(int32_t page_size, int32_t n_pages, int32_t n_seqs, const int32_t* q_len, const int32_t* kv_len, const int32_t* page_table, int32_t table_stride,
                int32_t max_tokens, int32_t max_pages, BatchTotals* totals, const char** why);

}  // namespace ggr
