// Page lookups of one decode step over a paged bank cache, made by
// resolve_kernel (pages.hip) and read by the decode kernel (decode.hip).
#pragma once

#include "bdm_common.h"

namespace bdm {

struct PageTables {
    void *pool;
    const int32_t *source;  // [N, KW] page that a written bank is read from; -1: the sequence has none
    const int32_t *target;  // [N, KW] page that it is stored to; -1: none was free
    const int32_t *read;    // [N, KR] page of a read bank; -1: none
};

// What bdm_decode would refuse of a step over pages (decode.hip); nothing is refused behind it.
int check_decode_pages(const bdm_decode_args *a);
// The decode step over the pages: bdm_decode's kernel with its states addressed by `tables`.
int launch_decode_pages(const bdm_decode_args &a, const PageTables &tables, hipStream_t stream);

}  // namespace bdm
