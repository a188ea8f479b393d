// Launch wrappers of the paged history (history.cu).
#pragma once

#include <cstdint>

#include <cuda_runtime.h>

namespace cb {

// Records of ragged sequences (rows) in pages of page_len records.  Row r holds
// lengths[r] records; record i lies in page table[r][i / page_len].  refs[p] is the
// number of table entries that name page p; pages with none are free.
struct HistoryView
{
    char* pages;           // [nPages, pageLen] records of recordBytes
    int* table;            // [nRows, rowPages], -1 where unused
    int* lengths;          // [nRows]
    int* refs;             // [nPages]
    long long recordBytes;
    int nRows, rowPages, nPages, pageLen;
};

// counter: set to 0, or null.
cudaError_t launchHistoryFork(const HistoryView& from, const HistoryView& to, const long long* parents, int* counter,
                              cudaStream_t s);

long long historyAppendWorkspace(const HistoryView& h);
// records: nRows rows of recordBytes, recordStride bytes apart; mask: u8 [nRows] or
// null; dropped: counter of the records that found no place.
cudaError_t launchHistoryAppend(const HistoryView& h, const char* records, long long recordStride, const uint8_t* mask,
                                int* dropped, void* workspace, cudaStream_t s);

void launchHistoryFree(const HistoryView& h, const uint8_t* mask, cudaStream_t s);

long long historyCompactWorkspace(const HistoryView& h);
cudaError_t launchHistoryCompact(const HistoryView& h, int* live, void* workspace, cudaStream_t s);

// out: [n, steps] records; counts: [n].  rows: n row indices, or null for all rows.
void launchHistoryRead(const HistoryView& h, const long long* rows, int n, int steps, char* out, int* counts,
                       cudaStream_t s);

}  // namespace cb
