// Paged history: the records of ragged sequences in pages that forked sequences
// share, with copy on write.
//
// All bookkeeping is on the device and deterministic: pages are handed out lowest
// first to the needy rows in row order (two prefix sums, no order of atomics), and
// counts are integers.  The data moves are bound by memory bandwidth.
#include "history.cuh"

#include <algorithm>

namespace cb {

namespace {

using u64 = unsigned long long;

constexpr unsigned FULL = 0xffffffffu;
constexpr int THREADS = 256;
constexpr int CHUNK = 1024;  // rows or pages whose counts one block takes together

inline unsigned blocks(long long n, int t) { return (unsigned)((n + t - 1) / t); }

// The page of a table entry, or -1 where the table names none.
__device__ __forceinline__ int pageAt(const HistoryView& h, long long row, int col)
{
    const int p = h.table[row * h.rowPages + col];
    return p >= 0 && p < h.nPages ? p : -1;
}
__device__ __forceinline__ int usedColumns(const HistoryView& h, int length)
{
    const int used = length <= 0 ? 0 : (length - 1) / h.pageLen + 1;
    return used < h.rowPages ? used : h.rowPages;
}

// ---- fork -----------------------------------------------------------------------------

__global__ void __launch_bounds__(THREADS) forkKernel(HistoryView from, HistoryView to, const long long* parents)
{
    const long long i = blockIdx.x * (long long)THREADS + threadIdx.x;
    if (i >= (long long)to.nRows * to.rowPages) return;
    const int r = (int)(i / to.rowPages), col = (int)(i - (long long)r * to.rowPages);
    const long long parent = parents[r];
    const bool keep = parent >= 0 && parent < from.nRows;  // anything else empties the row
    const int length = keep ? from.lengths[parent] : 0;
    const int page = keep && col < usedColumns(from, length) ? pageAt(from, parent, col) : -1;
    to.table[i] = page;
    if (page >= 0) atomicAdd(&to.refs[page], 1);
    if (col == 0) to.lengths[r] = length;
}

// ---- append ---------------------------------------------------------------------------

enum RowKind : uint8_t { ROW_IDLE = 0, ROW_IN_PLACE, ROW_NEW_PAGE, ROW_COPY, ROW_FULL };

struct AppendWork
{
    u64* leader;      // [nPages] longest, then first, of the rows that share the page and append
    int* sharers;     // [nPages] how many those are
    int* rowNeeds;    // [row chunks + 1] pages needed, then their prefix sums
    int* pageFree;    // [page chunks + 1] free pages, then their prefix sums
    int* freeList;    // [nRows] the lowest free pages
    int* target;      // [nRows] page a record goes to, -1 for none
    int* source;      // [nRows] page whose records come with it, -1 for none
    uint8_t* kind;    // [nRows]
    int rowChunks, pageChunks;
};

__host__ __device__ inline long long alignUp(long long n) { return (n + 15) / 16 * 16; }

AppendWork planAppend(const HistoryView& h, void* base, long long* bytes, long long* zeroBytes)
{
    AppendWork w{};
    w.rowChunks = (int)blocks(h.nRows, CHUNK);
    w.pageChunks = (int)blocks(h.nPages, CHUNK);
    char* c = static_cast<char*>(base);
    long long at = 0;
    auto take = [&](long long n) { const long long o = at; at += alignUp(n); return c + o; };
    w.leader = reinterpret_cast<u64*>(take(8ll * h.nPages));
    w.sharers = reinterpret_cast<int*>(take(4ll * h.nPages));
    if (zeroBytes) *zeroBytes = at;
    w.rowNeeds = reinterpret_cast<int*>(take(4ll * (w.rowChunks + 1)));
    w.pageFree = reinterpret_cast<int*>(take(4ll * (w.pageChunks + 1)));
    w.freeList = reinterpret_cast<int*>(take(4ll * h.nRows));
    w.target = reinterpret_cast<int*>(take(4ll * h.nRows));
    w.source = reinterpret_cast<int*>(take(4ll * h.nRows));
    w.kind = reinterpret_cast<uint8_t*>(take(h.nRows));
    if (bytes) *bytes = at;
    return w;
}

__device__ __forceinline__ u64 leaderKey(int slot, int row) { return (u64)(unsigned)slot << 32 | (unsigned)~row; }

// Whether a row appends, and where: page column, slot, and the page that holds the
// records before it (-1 at a page's start).
struct Append
{
    bool on, room;
    int col, slot, held;
};

__device__ __forceinline__ Append appendOf(const HistoryView& h, const uint8_t* mask, int r)
{
    Append a{};
    a.held = -1;
    a.on = !mask || mask[r];
    const int length = h.lengths[r];
    a.col = length / h.pageLen;
    a.slot = length - a.col * h.pageLen;
    a.room = length >= 0 && a.col < h.rowPages;
    if (a.on && a.room && a.slot > 0)
    {
        a.held = pageAt(h, r, a.col);
        a.room = a.held >= 0;
    }
    return a;
}

__global__ void __launch_bounds__(THREADS) appendShareKernel(HistoryView h, const uint8_t* mask, AppendWork w)
{
    const int r = (int)(blockIdx.x * (long long)THREADS + threadIdx.x);
    if (r >= h.nRows) return;
    const Append a = appendOf(h, mask, r);
    if (!a.on || a.held < 0 || h.refs[a.held] <= 1) return;
    atomicAdd(&w.sharers[a.held], 1);
    atomicMax(&w.leader[a.held], leaderKey(a.slot, r));
}

__device__ __forceinline__ int blockSum(int v)
{
    __shared__ int part[THREADS / 32];
    v = __reduce_add_sync(FULL, v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    int s = 0;
    for (int k = 0; k < THREADS / 32; k++) s += part[k];
    return s;
}

// Exclusive prefix sum of a flag over the block's threads; total over the block.
__device__ __forceinline__ int blockRank(bool flag, int& total)
{
    __shared__ int part[THREADS / 32];
    const unsigned votes = __ballot_sync(FULL, flag);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = __popc(votes);
    __syncthreads();
    int before = 0;
    total = 0;
    for (int k = 0; k < THREADS / 32; k++)
    {
        if (k < (int)(threadIdx.x >> 5)) before += part[k];
        total += part[k];
    }
    return before + __popc(votes & ((1u << (threadIdx.x & 31)) - 1));
}

// What each row needs, counted per chunk of rows; free pages per chunk of pages.
__global__ void __launch_bounds__(THREADS) appendCountKernel(HistoryView h, const uint8_t* mask, AppendWork w)
{
    const int b = blockIdx.x;
    int count = 0;
    if (b < w.rowChunks)
    {
        for (int i = threadIdx.x; i < CHUNK; i += THREADS)
        {
            const long long r = (long long)b * CHUNK + i;
            if (r >= h.nRows) break;
            const Append a = appendOf(h, mask, (int)r);
            RowKind kind = ROW_IDLE;
            if (a.on && !a.room)
                kind = ROW_FULL;
            else if (a.on && a.slot == 0)
                kind = ROW_NEW_PAGE;
            else if (a.on)
            {
                const int refs = h.refs[a.held];
                const bool stays = refs <= 1 || (w.sharers[a.held] == refs && w.leader[a.held] == leaderKey(a.slot, (int)r));
                kind = stays ? ROW_IN_PLACE : ROW_COPY;
            }
            w.kind[r] = kind;
            count += kind == ROW_NEW_PAGE || kind == ROW_COPY;
        }
        count = blockSum(count);
        if (threadIdx.x == 0) w.rowNeeds[b] = count;
    }
    else
    {
        const int c = b - w.rowChunks;
        for (int i = threadIdx.x; i < CHUNK; i += THREADS)
        {
            const long long p = (long long)c * CHUNK + i;
            if (p < h.nPages) count += h.refs[p] <= 0;
        }
        count = blockSum(count);
        if (threadIdx.x == 0) w.pageFree[c] = count;
    }
}

// Exclusive prefix sums of n counts in place, the total behind them; one block.
__device__ void scanCounts(int* counts, int n)
{
    __shared__ int part[THREADS];
    const int each = (n + THREADS - 1) / THREADS, i0 = threadIdx.x * each, i1 = min(n, i0 + each);
    int s = 0;
    for (int i = i0; i < i1; i++) s += counts[i];
    __syncthreads();
    part[threadIdx.x] = s;
    __syncthreads();
    int before = 0, total = 0;
    for (int k = 0; k < THREADS; k++)
    {
        if (k < (int)threadIdx.x) before += part[k];
        total += part[k];
    }
    for (int i = i0; i < i1; i++)
    {
        const int c = counts[i];
        counts[i] = before;
        before += c;
    }
    if (threadIdx.x == 0) counts[n] = total;
}

__global__ void __launch_bounds__(THREADS) scanKernel(int* a, int na, int* b, int nb)
{
    if (blockIdx.x == 0)
        scanCounts(a, na);
    else
        scanCounts(b, nb);
}

// The k-th free page for every k that a row needs.
__global__ void __launch_bounds__(THREADS) freeListKernel(HistoryView h, AppendWork w)
{
    const int needs = w.rowNeeds[w.rowChunks];
    int rank = w.pageFree[blockIdx.x];
    if (rank >= needs) return;
    for (int i0 = 0; i0 < CHUNK; i0 += THREADS)
    {
        const long long p = (long long)blockIdx.x * CHUNK + i0 + threadIdx.x;
        const bool isFree = p < h.nPages && h.refs[p] <= 0;
        int total;
        const int k = rank + blockRank(isFree, total);
        if (isFree && k < needs) w.freeList[k] = (int)p;
        rank += total;
    }
}

// Every row's page: table, counts and lengths; rows that find none are dropped.
__global__ void __launch_bounds__(THREADS) appendAssignKernel(HistoryView h, AppendWork w, int* dropped)
{
    const int nFree = w.pageFree[w.pageChunks];
    int rank = w.rowNeeds[blockIdx.x];
    for (int i0 = 0; i0 < CHUNK; i0 += THREADS)
    {
        const long long r = (long long)blockIdx.x * CHUNK + i0 + threadIdx.x;
        const RowKind kind = r < h.nRows ? (RowKind)w.kind[r] : ROW_IDLE;
        const bool needs = kind == ROW_NEW_PAGE || kind == ROW_COPY;
        int total;
        const int k = rank + blockRank(needs, total);
        rank += total;
        if (r >= h.nRows) continue;
        int target = -1, source = -1;
        const int length = h.lengths[r];
        const int col = length / h.pageLen;
        if (kind == ROW_IN_PLACE) target = h.table[r * h.rowPages + col];
        if (needs && k < nFree)
        {
            target = w.freeList[k];
            if (kind == ROW_COPY)
            {
                source = h.table[r * h.rowPages + col];
                atomicSub(&h.refs[source], 1);
            }
            h.refs[target] = 1;
            h.table[r * h.rowPages + col] = target;
        }
        if (target >= 0)
            h.lengths[r] = length + 1;
        else if (kind != ROW_IDLE)
            atomicAdd(dropped, 1);
        w.target[r] = target;
        w.source[r] = source;
    }
}

template <class U>
__device__ __forceinline__ void copyUnits(char* to, const char* from, long long bytes, int lane, int lanes)
{
    U* t = reinterpret_cast<U*>(to);
    const U* f = reinterpret_cast<const U*>(from);
    for (long long i = lane; i < bytes / (long long)sizeof(U); i += lanes) t[i] = f[i];
}

__device__ __forceinline__ void copyRecord(char* to, const char* from, long long bytes, int unit, int lane, int lanes)
{
    switch (unit)
    {
    case 16: copyUnits<uint4>(to, from, bytes, lane, lanes); break;
    case 8: copyUnits<uint2>(to, from, bytes, lane, lanes); break;
    case 4: copyUnits<unsigned>(to, from, bytes, lane, lanes); break;
    case 2: copyUnits<unsigned short>(to, from, bytes, lane, lanes); break;
    default: copyUnits<uint8_t>(to, from, bytes, lane, lanes); break;
    }
}

// A warp per (row, slot): the row's record, or one record of the page it copies.
__global__ void __launch_bounds__(THREADS) appendDataKernel(HistoryView h, AppendWork w, const char* records,
                                                            long long recordStride, int unit)
{
    const long long item = (blockIdx.x * (long long)THREADS + threadIdx.x) >> 5;
    const int lane = threadIdx.x & 31;
    const long long r = item / h.pageLen;
    const int s = (int)(item - r * h.pageLen);
    if (r >= h.nRows) return;
    const int target = w.target[r];
    if (target < 0) return;
    const int slot = (h.lengths[r] - 1) % h.pageLen;
    const int source = w.source[r];
    char* to = h.pages + ((long long)target * h.pageLen + s) * h.recordBytes;
    if (s == slot)
        copyRecord(to, records + r * recordStride, h.recordBytes, unit, lane, 32);
    else if (s < slot && source >= 0)
        copyRecord(to, h.pages + ((long long)source * h.pageLen + s) * h.recordBytes, h.recordBytes, unit, lane, 32);
}

// ---- free -----------------------------------------------------------------------------

__global__ void __launch_bounds__(THREADS) freeKernel(HistoryView h, const uint8_t* mask)
{
    const long long i = blockIdx.x * (long long)THREADS + threadIdx.x;
    if (i >= (long long)h.nRows * h.rowPages) return;
    const int r = (int)(i / h.rowPages);
    if (!mask[r]) return;
    const int col = (int)(i - (long long)r * h.rowPages);
    const int page = pageAt(h, r, col);
    if (page >= 0) atomicSub(&h.refs[page], 1);
    h.table[i] = -1;
    if (col == 0) h.lengths[r] = 0;
}

// ---- compact --------------------------------------------------------------------------

struct CompactWork
{
    int* liveCount;   // [page chunks + 1]
    int* hole;        // [nPages] hole of rank k
    int* moved;       // [nPages] page that goes to hole k
    int* rankOf;      // [nPages] k of a page that moves
    int pageChunks;
};

CompactWork planCompact(const HistoryView& h, void* base, long long* bytes)
{
    CompactWork w{};
    w.pageChunks = (int)blocks(h.nPages, CHUNK);
    char* c = static_cast<char*>(base);
    long long at = 0;
    auto take = [&](long long n) { const long long o = at; at += alignUp(n); return reinterpret_cast<int*>(c + o); };
    w.liveCount = take(4ll * (w.pageChunks + 1));
    w.hole = take(4ll * h.nPages);
    w.moved = take(4ll * h.nPages);
    w.rankOf = take(4ll * h.nPages);
    if (bytes) *bytes = at;
    return w;
}

__global__ void __launch_bounds__(THREADS) liveCountKernel(HistoryView h, CompactWork w)
{
    int count = 0;
    for (int i = threadIdx.x; i < CHUNK; i += THREADS)
    {
        const long long p = (long long)blockIdx.x * CHUNK + i;
        if (p < h.nPages) count += h.refs[p] > 0;
    }
    count = blockSum(count);
    if (threadIdx.x == 0) w.liveCount[blockIdx.x] = count;
}

// With L live pages, the k-th hole below L takes the k-th highest live page: both
// ranks come from the number of live pages before a page.
__global__ void __launch_bounds__(THREADS) compactPlanKernel(HistoryView h, CompactWork w, int* live)
{
    const int L = w.liveCount[w.pageChunks];
    if (blockIdx.x == 0 && threadIdx.x == 0) *live = L;
    int before = w.liveCount[blockIdx.x];
    for (int i0 = 0; i0 < CHUNK; i0 += THREADS)
    {
        const long long p = (long long)blockIdx.x * CHUNK + i0 + threadIdx.x;
        const bool isLive = p < h.nPages && h.refs[p] > 0;
        int total;
        const int q = before + blockRank(isLive, total);
        before += total;
        if (p >= h.nPages) continue;
        if (!isLive && p < L) w.hole[p - q] = (int)p;
        if (isLive && p >= L)
        {
            w.moved[L - 1 - q] = (int)p;
            w.rankOf[p] = L - 1 - q;
        }
    }
}

__global__ void __launch_bounds__(THREADS) compactTableKernel(HistoryView h, CompactWork w)
{
    const long long i = blockIdx.x * (long long)THREADS + threadIdx.x;
    if (i >= (long long)h.nRows * h.rowPages) return;
    const int page = h.table[i], L = w.liveCount[w.pageChunks];
    if (page >= L && page < h.nPages && h.refs[page] > 0) h.table[i] = w.hole[w.rankOf[page]];
}

// Blocks take the moves in turn; their number is known on the device only.
__global__ void __launch_bounds__(THREADS) compactMoveKernel(HistoryView h, CompactWork w, int unit)
{
    const int L = w.liveCount[w.pageChunks];
    // Live pages at or beyond L, as many as there are holes below it.
    const long long bytes = (long long)h.pageLen * h.recordBytes;
    for (int k = blockIdx.x; k < h.nPages - L && k < L; k += gridDim.x)
    {
        const int to = w.hole[k], from = w.moved[k];
        if (from < 0) break;
        copyRecord(h.pages + to * bytes, h.pages + from * bytes, bytes, unit, threadIdx.x, THREADS);
        if (threadIdx.x == 0)
        {
            h.refs[to] = h.refs[from];
            h.refs[from] = 0;
        }
    }
}

// ---- read -----------------------------------------------------------------------------

// A warp per (row, step): the last min(length, steps) records of a row, zeros behind.
__global__ void __launch_bounds__(THREADS) readKernel(HistoryView h, const long long* rows, int n, int steps, char* out,
                                                      int* counts, int unit)
{
    const long long item = (blockIdx.x * (long long)THREADS + threadIdx.x) >> 5;
    const int lane = threadIdx.x & 31;
    const long long i = item / steps;
    const int t = (int)(item - i * steps);
    if (i >= n) return;
    const long long r = rows ? rows[i] : i;
    int length = r >= 0 && r < h.nRows ? h.lengths[r] : 0;
    length = max(0, min(length, (int)min((long long)h.rowPages * h.pageLen, 0x7fffffffll)));
    const int count = min(length, steps);
    if (t == 0 && lane == 0) counts[i] = count;
    char* to = out + item * h.recordBytes;
    int page = -1, at = 0;
    if (t < count)
    {
        at = length - count + t;
        page = pageAt(h, r, at / h.pageLen);
    }
    if (page >= 0)
    {
        copyRecord(to, h.pages + ((long long)page * h.pageLen + at % h.pageLen) * h.recordBytes, h.recordBytes, unit,
                   lane, 32);
        return;
    }
    for (long long b = lane; b < h.recordBytes; b += 32) to[b] = 0;
}

int unitOf(unsigned long long bits)
{
    int unit = 16;
    while (bits % unit) unit /= 2;
    return unit;
}

}  // namespace

cudaError_t launchHistoryFork(const HistoryView& from, const HistoryView& to, const long long* parents, cudaStream_t s)
{
    if (to.nPages > 0)
    {
        const cudaError_t err = cudaMemsetAsync(to.refs, 0, 4ll * to.nPages, s);
        if (err != cudaSuccess) return err;
    }
    const long long n = (long long)to.nRows * to.rowPages;
    if (n > 0) forkKernel<<<blocks(n, THREADS), THREADS, 0, s>>>(from, to, parents);
    return cudaGetLastError();
}

long long historyAppendWorkspace(const HistoryView& h)
{
    long long bytes = 0;
    planAppend(h, nullptr, &bytes, nullptr);
    return bytes;
}

cudaError_t launchHistoryAppend(const HistoryView& h, const char* records, long long recordStride, const uint8_t* mask,
                                int* dropped, void* workspace, cudaStream_t s)
{
    if (h.nRows == 0) return cudaSuccess;
    long long zero = 0;
    const AppendWork w = planAppend(h, workspace, nullptr, &zero);
    if (zero > 0)
    {
        const cudaError_t err = cudaMemsetAsync(workspace, 0, zero, s);
        if (err != cudaSuccess) return err;
    }
    appendShareKernel<<<blocks(h.nRows, THREADS), THREADS, 0, s>>>(h, mask, w);
    appendCountKernel<<<w.rowChunks + w.pageChunks, THREADS, 0, s>>>(h, mask, w);
    scanKernel<<<2, THREADS, 0, s>>>(w.rowNeeds, w.rowChunks, w.pageFree, w.pageChunks);
    if (w.pageChunks > 0) freeListKernel<<<w.pageChunks, THREADS, 0, s>>>(h, w);
    appendAssignKernel<<<w.rowChunks, THREADS, 0, s>>>(h, w, dropped);
    const int unit = unitOf(reinterpret_cast<uintptr_t>(h.pages) | reinterpret_cast<uintptr_t>(records)
                            | (unsigned long long)h.recordBytes | (unsigned long long)recordStride);
    appendDataKernel<<<blocks((long long)h.nRows * h.pageLen * 32, THREADS), THREADS, 0, s>>>(h, w, records, recordStride,
                                                                                             unit);
    return cudaGetLastError();
}

void launchHistoryFree(const HistoryView& h, const uint8_t* mask, cudaStream_t s)
{
    const long long n = (long long)h.nRows * h.rowPages;
    if (n > 0) freeKernel<<<blocks(n, THREADS), THREADS, 0, s>>>(h, mask);
}

long long historyCompactWorkspace(const HistoryView& h)
{
    long long bytes = 0;
    planCompact(h, nullptr, &bytes);
    return bytes;
}

cudaError_t launchHistoryCompact(const HistoryView& h, int* live, void* workspace, cudaStream_t s)
{
    if (h.nPages == 0) return cudaMemsetAsync(live, 0, sizeof(int), s);
    const CompactWork w = planCompact(h, workspace, nullptr);
    // -1 marks the end of the moves.
    const cudaError_t err = cudaMemsetAsync(w.moved, 0xff, 4ll * h.nPages, s);
    if (err != cudaSuccess) return err;
    liveCountKernel<<<w.pageChunks, THREADS, 0, s>>>(h, w);
    scanKernel<<<1, THREADS, 0, s>>>(w.liveCount, w.pageChunks, nullptr, 0);
    compactPlanKernel<<<w.pageChunks, THREADS, 0, s>>>(h, w, live);
    const long long n = (long long)h.nRows * h.rowPages;
    if (n > 0) compactTableKernel<<<blocks(n, THREADS), THREADS, 0, s>>>(h, w);
    const int unit = unitOf(reinterpret_cast<uintptr_t>(h.pages) | (unsigned long long)h.recordBytes * h.pageLen);
    compactMoveKernel<<<(unsigned)std::min(h.nPages, 148 * 8), THREADS, 0, s>>>(h, w, unit);
    return cudaGetLastError();
}

void launchHistoryRead(const HistoryView& h, const long long* rows, int n, int steps, char* out, int* counts,
                       cudaStream_t s)
{
    if (n <= 0 || steps <= 0) return;
    const int unit = unitOf(reinterpret_cast<uintptr_t>(h.pages) | reinterpret_cast<uintptr_t>(out)
                            | (unsigned long long)h.recordBytes);
    readKernel<<<blocks((long long)n * steps * 32, THREADS), THREADS, 0, s>>>(h, rows, n, steps, out, counts, unit);
}

}  // namespace cb
