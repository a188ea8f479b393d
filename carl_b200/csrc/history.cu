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
constexpr int CHUNK = THREADS;          // rows or pages that one block counts
constexpr int ITEM_BYTES = 4096;        // what a warp copies, where records are smaller

inline unsigned blocks(long long n, int t) { return (unsigned)((n + t - 1) / t); }

// ---- copies of whole records -------------------------------------------------------------

// Copies `bytes` with the threads of a warp or block (tid of `threads`); four loads of a
// thread are under way before the first store.
template <class U>
__device__ __forceinline__ void copyUnits(char* to, const char* from, long long bytes, int tid, int threads)
{
    U* t = reinterpret_cast<U*>(to);
    const U* f = reinterpret_cast<const U*>(from);
    const long long n = bytes / (long long)sizeof(U);
    long long i = tid;
    for (; i + 3ll * threads < n; i += 4ll * threads)
    {
        U v[4];
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = f[i + (long long)k * threads];
#pragma unroll
        for (int k = 0; k < 4; k++) t[i + (long long)k * threads] = v[k];
    }
    U v[3];
#pragma unroll
    for (int k = 0; k < 3; k++)
        if (i + (long long)k * threads < n) v[k] = f[i + (long long)k * threads];
#pragma unroll
    for (int k = 0; k < 3; k++)
        if (i + (long long)k * threads < n) t[i + (long long)k * threads] = v[k];
}

__device__ __forceinline__ void copyBytes(char* to, const char* from, long long bytes, int unit, int tid, int threads)
{
    switch (unit)
    {
    case 16: copyUnits<uint4>(to, from, bytes, tid, threads); break;
    case 8: copyUnits<uint2>(to, from, bytes, tid, threads); break;
    case 4: copyUnits<unsigned>(to, from, bytes, tid, threads); break;
    case 2: copyUnits<unsigned short>(to, from, bytes, tid, threads); break;
    default: copyUnits<uint8_t>(to, from, bytes, tid, threads); break;
    }
}

// Largest unit that divides addresses and sizes (their bits or-ed together).
int unitOf(unsigned long long bits)
{
    int unit = 16;
    while (bits % unit) unit /= 2;
    return unit;
}

// Records of an item of work.
int itemRecords(long long recordBytes, int most)
{
    return (int)std::max<long long>(1, std::min<long long>(most, ITEM_BYTES / recordBytes));
}

// ---- counts ------------------------------------------------------------------------------

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

// Entry i of the forked table, and with the first of a row its length.
__device__ __forceinline__ void forkEntry(const HistoryView& from, const HistoryView& to, const long long* parents, long long i)
{
    const int r = (int)(i / to.rowPages), col = (int)(i - (long long)r * to.rowPages);
    const long long parent = parents[r];
    const bool keep = parent >= 0 && parent < from.nRows;  // anything else empties the row
    const int length = keep ? from.lengths[parent] : 0;
    const int page = keep && col < usedColumns(from, length) ? pageAt(from, parent, col) : -1;
    to.table[i] = page;
    if (page >= 0) atomicAdd(&to.refs[page], 1);
    if (col == 0) to.lengths[r] = length;
}

__global__ void __launch_bounds__(THREADS) forkKernel(HistoryView from, HistoryView to, const long long* parents, int* counter)
{
    const long long i = blockIdx.x * (long long)THREADS + threadIdx.x;
    if (i == 0 && counter) *counter = 0;
    if (i < (long long)to.nRows * to.rowPages) forkEntry(from, to, parents, i);
}

// Small histories: every kernel of an operator that only keeps the books, in one block, so
// that a call is one or two launches instead of up to four (8 rows of 8 pages, forked and
// appended to: 16 us on the device in seven launches, 9 us in two).
constexpr int SMALL_THREADS = 1024;
constexpr int SMALL_PAGES = 16 * 1024;     // pages, and table entries
constexpr int SMALL_ROWS = SMALL_THREADS;  // rows of an append, one a thread
constexpr long long SMALL_COPY = 512 * 1024;  // most that one SM copies in an append, bytes

__global__ void __launch_bounds__(SMALL_THREADS) forkSmallKernel(HistoryView from, HistoryView to, const long long* parents,
                                                                 int* counter)
{
    for (int p = threadIdx.x; p < to.nPages; p += SMALL_THREADS) to.refs[p] = 0;
    if (threadIdx.x == 0 && counter) *counter = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < to.nRows * to.rowPages; i += SMALL_THREADS) forkEntry(from, to, parents, i);
}

// ---- append ---------------------------------------------------------------------------

// What a row needs, from the counts before anything changes.
enum RowKind { ROW_IDLE = 0, ROW_IN_PLACE, ROW_NEW_PAGE, ROW_COPY, ROW_FULL };

struct Job
{
    int kind;
    int length;  // before the record
    int held;    // page with the records before it, -1 at a page's start
    int rank;    // rows in need before it in its chunk
};

struct AppendWork
{
    u64* leader;      // [nPages] longest, then first, of the rows that share the page and append
    int* sharers;     // [nPages] how many those are
    unsigned* done;   // blocks that have counted
    int* rowNeeds;    // [row chunks + 1] pages needed, then their prefix sums
    int* pageFree;    // [page chunks + 1] free pages, then their prefix sums
    unsigned* bits;   // [page chunks, CHUNK / 32] free pages
    Job* job;         // [nRows]
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
    w.done = reinterpret_cast<unsigned*>(take(4));
    w.leader = reinterpret_cast<u64*>(take(8ll * h.nPages));
    w.sharers = reinterpret_cast<int*>(take(4ll * h.nPages));
    if (zeroBytes) *zeroBytes = at;
    w.rowNeeds = reinterpret_cast<int*>(take(4ll * (w.rowChunks + 1)));
    w.pageFree = reinterpret_cast<int*>(take(4ll * (w.pageChunks + 1)));
    w.bits = reinterpret_cast<unsigned*>(take(4ll * w.pageChunks * (CHUNK / 32)));
    w.job = reinterpret_cast<Job*>(take((long long)sizeof(Job) * h.nRows));
    if (bytes) *bytes = at;
    return w;
}

__device__ __forceinline__ u64 leaderKey(int slot, int row) { return (u64)(unsigned)slot << 32 | (unsigned)~row; }

// Whether a row appends, and where: page column, slot, and the page that holds the
// records before it (-1 at a page's start).
struct Append
{
    bool on, room;
    int length, col, slot, held;
};

__device__ __forceinline__ Append appendOf(const HistoryView& h, const uint8_t* mask, int r)
{
    Append a{};
    a.held = -1;
    a.on = !mask || mask[r];
    a.length = h.lengths[r];
    a.col = a.length / h.pageLen;
    a.slot = a.length - a.col * h.pageLen;
    a.room = a.length >= 0 && a.col < h.rowPages;
    if (a.on && a.room && a.slot > 0)
    {
        a.held = pageAt(h, r, a.col);
        a.room = a.held >= 0;
    }
    return a;
}

__device__ __forceinline__ void share(const HistoryView& h, const uint8_t* mask, const AppendWork& w, int r)
{
    if (r >= h.nRows) return;
    const Append a = appendOf(h, mask, r);
    if (!a.on || a.held < 0 || h.refs[a.held] <= 1) return;
    atomicAdd(&w.sharers[a.held], 1);
    atomicMax(&w.leader[a.held], leaderKey(a.slot, r));
}

__global__ void __launch_bounds__(THREADS) appendShareKernel(HistoryView h, const uint8_t* mask, AppendWork w)
{
    share(h, mask, w, (int)min(blockIdx.x * (long long)THREADS + threadIdx.x, (long long)h.nRows));
}

// Exclusive prefix sum of a flag over the block's threads; total over the block.
template <int N = THREADS>
__device__ __forceinline__ int blockRank(bool flag, int& total)
{
    __shared__ int part[N / 32];
    const unsigned votes = __ballot_sync(FULL, flag);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = __popc(votes);
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int k = 0; k < N / 32; k++)
    {
        if (k < (int)(threadIdx.x >> 5)) before += part[k];
        total += part[k];
    }
    return before + __popc(votes & ((1u << (threadIdx.x & 31)) - 1));
}

// Exclusive prefix sums of n counts in place, the total behind them; one block.
__device__ void scanCounts(int* counts, int n)
{
    __shared__ int part[THREADS / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int carry = 0;
    for (int i0 = 0; i0 < n; i0 += THREADS)
    {
        const int i = i0 + threadIdx.x, mine = i < n ? __ldcg(counts + i) : 0;
        int sum = mine;
#pragma unroll
        for (int d = 1; d < 32; d *= 2)
        {
            const int o = __shfl_up_sync(FULL, sum, d);
            if (lane >= d) sum += o;
        }
        __syncthreads();
        if (lane == 31) part[warp] = sum;
        __syncthreads();
        int total = 0;
#pragma unroll
        for (int k = 0; k < THREADS / 32; k++)
        {
            if (k < warp) sum += part[k];
            total += part[k];
        }
        if (i < n) counts[i] = carry + sum - mine;
        carry += total;
    }
    if (threadIdx.x == 0) counts[n] = carry;
}

// Whether this block is the last to come here; what the others wrote before is visible.
__device__ __forceinline__ bool lastBlock(unsigned* done)
{
    __shared__ bool last;
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) last = atomicAdd(done, 1) + 1 == gridDim.x;
    __syncthreads();
    if (last) __threadfence();
    return last;
}

// What a row needs (but for its rank), once the sharers are known.
__device__ __forceinline__ Job jobOf(const HistoryView& h, const uint8_t* mask, const AppendWork& w, int r)
{
    Job job{ ROW_IDLE, 0, -1, 0 };
    if (r >= h.nRows) return job;
    const Append a = appendOf(h, mask, r);
    job.length = a.length;
    job.held = a.held;
    if (a.on && !a.room)
        job.kind = ROW_FULL;
    else if (a.on && a.slot == 0)
        job.kind = ROW_NEW_PAGE;
    else if (a.on)
    {
        const int refs = h.refs[a.held];
        const bool stays = refs <= 1 || (w.sharers[a.held] == refs && w.leader[a.held] == leaderKey(a.slot, r));
        job.kind = stays ? ROW_IN_PLACE : ROW_COPY;
    }
    return job;
}

// What each row needs, counted per chunk of rows; the free pages, counted per chunk of
// pages.  The last block adds the counts up.
__global__ void __launch_bounds__(THREADS) appendCountKernel(HistoryView h, const uint8_t* mask, AppendWork w)
{
    const int b = blockIdx.x;
    int total;
    if (b < w.rowChunks)
    {
        const long long r = (long long)b * CHUNK + threadIdx.x;
        Job job = jobOf(h, mask, w, (int)min(r, (long long)h.nRows));
        job.rank = blockRank(job.kind == ROW_NEW_PAGE || job.kind == ROW_COPY, total);
        if (r < h.nRows) w.job[r] = job;
        if (threadIdx.x == 0) w.rowNeeds[b] = total;
    }
    else
    {
        const int c = b - w.rowChunks;
        const long long p = (long long)c * CHUNK + threadIdx.x;
        const bool isFree = p < h.nPages && h.refs[p] <= 0;
        const unsigned votes = __ballot_sync(FULL, isFree);
        if ((threadIdx.x & 31) == 0) w.bits[c * (CHUNK / 32) + (threadIdx.x >> 5)] = votes;
        blockRank(isFree, total);
        if (threadIdx.x == 0) w.pageFree[c] = total;
    }
    if (!lastBlock(w.done)) return;
    scanCounts(w.rowNeeds, w.rowChunks);
    __syncthreads();
    scanCounts(w.pageFree, w.pageChunks);
}

// The k-th free page: its chunk by bisection of the prefix sums, then its bit.
__device__ __forceinline__ int freePage(const AppendWork& w, int k)
{
    int lo = 0, hi = w.pageChunks - 1;
    while (lo < hi)
    {
        const int mid = (lo + hi + 1) / 2;
        if (w.pageFree[mid] <= k)
            lo = mid;
        else
            hi = mid - 1;
    }
    k -= w.pageFree[lo];
    const uint4* bits = reinterpret_cast<const uint4*>(w.bits + lo * (CHUNK / 32));
    const uint4 a = bits[0], b = bits[1];
    const unsigned word[CHUNK / 32] = { a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w };
    int page = lo * CHUNK;
#pragma unroll
    for (int i = 0; i < CHUNK / 32; i++)
    {
        const int n = __popc(word[i]);
        if (k >= 0 && k < n) return page + 32 * i + __fns(word[i], 0, k + 1);
        k -= n;
    }
    return -1;
}

// A warp per row and item of its page: the records that come along with a copied page,
// and the row's own.  16384 rows of 1008-byte records, a third of them copying 7.5 records,
// move 117 MB in 33 us, 54 % of the copy rate; a warp per record took 53.  Bound by latency:
// before its first byte a warp follows the row's job, the prefix sums, a bisection for the free
// page and its bits, one load after another.  The first item's warp enters the row's page and
// length.
__global__ void __launch_bounds__(THREADS) appendWriteKernel(HistoryView h, AppendWork w, const char* records,
                                                             long long recordStride, int unit, int perItem, int items,
                                                             int* dropped)
{
    const long long item = (blockIdx.x * (long long)THREADS + threadIdx.x) >> 5;
    const int lane = threadIdx.x & 31;
    const long long r = item / items;
    if (r >= h.nRows) return;
    const int part = (int)(item - r * items);
    const int4 j = *reinterpret_cast<const int4*>(w.job + r);
    const Job job{ j.x, j.y, j.z, j.w };
    if (job.kind == ROW_IDLE) return;
    const int col = job.length / h.pageLen, slot = job.length - col * h.pageLen;
    const int s0 = part * perItem, s1 = s0 + min(perItem, slot - s0);  // s0 + perItem may pass 2^31
    const bool own = s0 <= slot && slot - s0 < perItem, copies = job.kind == ROW_COPY && s0 < s1;
    if (!own && !copies && part != 0) return;
    int target = job.kind == ROW_IN_PLACE ? job.held : -1;
    if (job.kind == ROW_NEW_PAGE || job.kind == ROW_COPY)
    {
        const int k = w.rowNeeds[r / CHUNK] + job.rank;
        if (k < w.pageFree[w.pageChunks]) target = freePage(w, k);
    }
    if (part == 0 && lane == 0)
    {
        if (target < 0)
            atomicAdd(dropped, 1);
        else
        {
            h.lengths[r] = job.length + 1;
            if (job.kind != ROW_IN_PLACE)
            {
                h.table[r * h.rowPages + col] = target;
                h.refs[target] = 1;
                if (job.kind == ROW_COPY) atomicSub(&h.refs[job.held], 1);
            }
        }
    }
    if (target < 0) return;
    char* to = h.pages + (long long)target * h.pageLen * h.recordBytes;
    if (copies)
        copyBytes(to + s0 * h.recordBytes, h.pages + ((long long)job.held * h.pageLen + s0) * h.recordBytes,
                  (s1 - s0) * h.recordBytes, unit, lane, 32);
    if (own) copyBytes(to + slot * h.recordBytes, records + r * recordStride, h.recordBytes, unit, lane, 32);
}

__global__ void __launch_bounds__(SMALL_THREADS) appendSmallKernel(HistoryView h, const uint8_t* mask, AppendWork w,
                                                                   const char* records, long long recordStride, int unit,
                                                                   int perItem, int items, int* dropped)
{
    __shared__ int freeS[SMALL_ROWS], targetS[SMALL_ROWS], lengthS[SMALL_ROWS], sourceS[SMALL_ROWS];
    const int r = threadIdx.x, lane = r & 31;
    for (int p = r; p < h.nPages; p += SMALL_THREADS)
    {
        w.leader[p] = 0;
        w.sharers[p] = 0;
    }
    __syncthreads();
    share(h, mask, w, min(r, h.nRows));
    __syncthreads();
    const Job job = jobOf(h, mask, w, min(r, h.nRows));
    int needs, found = 0;
    const bool need = job.kind == ROW_NEW_PAGE || job.kind == ROW_COPY;
    const int rank = blockRank<SMALL_THREADS>(need, needs);
    for (int p0 = 0; p0 < h.nPages && found < needs; p0 += SMALL_THREADS)  // the same for all threads
    {
        const int p = p0 + r;
        const bool isFree = p < h.nPages && h.refs[p] <= 0;
        int total;
        const int k = found + blockRank<SMALL_THREADS>(isFree, total);
        if (isFree && k < needs) freeS[k] = p;
        found += total;
    }
    __syncthreads();
    int target = job.kind == ROW_IN_PLACE ? job.held : -1;
    if (need && rank < found) target = freeS[rank];
    targetS[r] = target;
    lengthS[r] = job.length;
    sourceS[r] = job.kind == ROW_COPY ? job.held : -1;
    if (r < h.nRows && job.kind != ROW_IDLE)
    {
        if (target < 0)
            atomicAdd(dropped, 1);
        else
        {
            h.lengths[r] = job.length + 1;
            if (need)
            {
                h.table[(long long)r * h.rowPages + job.length / h.pageLen] = target;
                h.refs[target] = 1;
                if (job.kind == ROW_COPY) atomicSub(&h.refs[job.held], 1);
            }
        }
    }
    __syncthreads();
    for (int i = r >> 5; i < h.nRows * items; i += SMALL_THREADS / 32)
    {
        const int row = i / items, s0 = (i - row * items) * perItem;
        if (targetS[row] < 0) continue;
        const int slot = lengthS[row] % h.pageLen, s1 = min(s0 + perItem, slot);
        char* to = h.pages + (long long)targetS[row] * h.pageLen * h.recordBytes;
        if (sourceS[row] >= 0 && s0 < s1)
            copyBytes(to + s0 * h.recordBytes, h.pages + ((long long)sourceS[row] * h.pageLen + s0) * h.recordBytes,
                      (s1 - s0) * h.recordBytes, unit, lane, 32);
        if (s0 <= slot && slot < s0 + perItem)
            copyBytes(to + slot * h.recordBytes, records + row * recordStride, h.recordBytes, unit, lane, 32);
    }
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
    unsigned* done;   // blocks that have counted
    int* moves;       // pages that move
    int* liveCount;   // [page chunks + 1]
    int* hole;        // [nPages] hole of rank k
    int* moved;       // [nPages] page that goes to hole k
    int* rankOf;      // [nPages] k of a page that moves, -1 of another
    int pageChunks;
};

CompactWork planCompact(const HistoryView& h, void* base, long long* bytes)
{
    CompactWork w{};
    w.pageChunks = (int)blocks(h.nPages, CHUNK);
    char* c = static_cast<char*>(base);
    long long at = 0;
    auto take = [&](long long n) { const long long o = at; at += alignUp(n); return reinterpret_cast<int*>(c + o); };
    w.done = reinterpret_cast<unsigned*>(take(4));
    w.moves = take(4);
    w.liveCount = take(4ll * (w.pageChunks + 1));
    w.hole = take(4ll * h.nPages);
    w.moved = take(4ll * h.nPages);
    w.rankOf = take(4ll * h.nPages);
    if (bytes) *bytes = at;
    return w;
}

__global__ void __launch_bounds__(THREADS) liveCountKernel(HistoryView h, CompactWork w, int* live)
{
    const long long p = (long long)blockIdx.x * CHUNK + threadIdx.x;
    int total;
    blockRank(p < h.nPages && h.refs[p] > 0, total);
    if (threadIdx.x == 0) w.liveCount[blockIdx.x] = total;
    if (!lastBlock(w.done)) return;
    scanCounts(w.liveCount, w.pageChunks);
    if (threadIdx.x == 0)
    {
        *live = w.liveCount[w.pageChunks];
        if (*live == h.nPages) *w.moves = 0;  // otherwise page L tells
    }
}

// With L live pages, the k-th hole below L takes the k-th highest live page: both ranks
// come from the number q of live pages before page p.
__device__ __forceinline__ void placePage(const CompactWork& w, int p, int q, bool isLive, int L)
{
    if (p == L) *w.moves = L - q;
    if (p < L)
    {
        if (!isLive) w.hole[p - q] = p;
        return;
    }
    w.rankOf[p] = isLive ? L - 1 - q : -1;
    if (isLive) w.moved[L - 1 - q] = p;
}

__global__ void __launch_bounds__(THREADS) compactPlanKernel(HistoryView h, CompactWork w)
{
    const int L = w.liveCount[w.pageChunks];
    const long long p = (long long)blockIdx.x * CHUNK + threadIdx.x;
    const bool isLive = p < h.nPages && h.refs[p] > 0;
    int total;
    const int q = w.liveCount[blockIdx.x] + blockRank(isLive, total);
    if (p < h.nPages) placePage(w, (int)p, q, isLive, L);
}

__global__ void __launch_bounds__(SMALL_THREADS) compactSmallKernel(HistoryView h, CompactWork w, int* live)
{
    int L = 0, total;
    for (int p0 = 0; p0 < h.nPages; p0 += SMALL_THREADS)
    {
        const int p = p0 + threadIdx.x;
        blockRank<SMALL_THREADS>(p < h.nPages && h.refs[p] > 0, total);
        L += total;
    }
    int before = 0;
    for (int p0 = 0; p0 < h.nPages; p0 += SMALL_THREADS)
    {
        const int p = p0 + threadIdx.x;
        const bool isLive = p < h.nPages && h.refs[p] > 0;
        const int q = before + blockRank<SMALL_THREADS>(isLive, total);
        before += total;
        if (p < h.nPages) placePage(w, p, q, isLive, L);
    }
    if (threadIdx.x == 0)
    {
        *live = w.liveCount[w.pageChunks] = L;
        if (L == h.nPages) *w.moves = 0;
    }
}

// The first blocks take the moves in turn (their number is known on the device only),
// the others follow them in the table.  Bound by memory: 4300 pages of 16 KB in 23 us.
__global__ void __launch_bounds__(THREADS) compactMoveKernel(HistoryView h, CompactWork w, int movers, int unit)
{
    const int L = w.liveCount[w.pageChunks];
    if ((int)blockIdx.x >= movers)
    {
        const long long i = (blockIdx.x - movers) * (long long)THREADS + threadIdx.x;
        if (i >= (long long)h.nRows * h.rowPages) return;
        const int page = h.table[i];
        if (page >= L && page < h.nPages && w.rankOf[page] >= 0) h.table[i] = w.hole[w.rankOf[page]];
        return;
    }
    const long long bytes = (long long)h.pageLen * h.recordBytes;
    const int moves = *w.moves;
    for (int k = blockIdx.x; k < moves; k += movers)
    {
        const int to = w.hole[k], from = w.moved[k];
        copyBytes(h.pages + to * bytes, h.pages + from * bytes, bytes, unit, threadIdx.x, THREADS);
        if (threadIdx.x == 0)
        {
            h.refs[to] = h.refs[from];
            h.refs[from] = 0;
        }
    }
}

// ---- read -----------------------------------------------------------------------------

// A warp per item of `perItem` steps of a row: the last min(length, steps) records of the
// row, zeros behind them.  Lane l finds record l of the item.  Bound by memory: 65536
// places of 1008 bytes written, the records among them read, in 21 us.
template <class U>
__global__ void __launch_bounds__(THREADS) readKernel(HistoryView h, const long long* rows, int n, int steps, int perItem,
                                                      int items, char* out, int* counts)
{
    const long long item = (blockIdx.x * (long long)THREADS + threadIdx.x) >> 5;
    const int lane = threadIdx.x & 31;
    const long long i = item / items;
    if (i >= n) return;
    const int part = (int)(item - i * items), t0 = part * perItem, here = min(perItem, steps - t0);
    const long long r = rows ? rows[i] : i;
    int length = r >= 0 && r < h.nRows ? h.lengths[r] : 0;
    length = (int)max(0ll, min((long long)length, (long long)h.rowPages * h.pageLen));
    const int count = min(length, steps);
    if (part == 0 && lane == 0) counts[i] = count;
    long long source = -1;  // record of the pages
    if (lane < here && t0 + lane < count)
    {
        const int at = length - count + t0 + lane, col = at / h.pageLen, page = pageAt(h, r, col);
        if (page >= 0) source = (long long)page * h.pageLen + at - col * h.pageLen;
    }
    const int units = (int)(h.recordBytes / sizeof(U)), all = here * units;
    U* to = reinterpret_cast<U*>(out + (i * steps + t0) * h.recordBytes);
    const U* pages = reinterpret_cast<const U*>(h.pages);
    constexpr int AHEAD = 4;
    for (int u0 = 0; u0 < all; u0 += 32 * AHEAD)
    {
        U v[AHEAD];
#pragma unroll
        for (int a = 0; a < AHEAD; a++)
        {
            const int u = u0 + 32 * a + lane, record = u / units;
            const long long from = __shfl_sync(FULL, source, record & 31);
            v[a] = U{};
            if (u < all && from >= 0) v[a] = pages[from * units + (u - record * units)];
        }
#pragma unroll
        for (int a = 0; a < AHEAD; a++)
            if (u0 + 32 * a + lane < all) to[u0 + 32 * a + lane] = v[a];
    }
}

}  // namespace

cudaError_t launchHistoryFork(const HistoryView& from, const HistoryView& to, const long long* parents, int* counter,
                              cudaStream_t s)
{
    const long long n = (long long)to.nRows * to.rowPages;
    if (n <= SMALL_PAGES && to.nPages <= SMALL_PAGES)
    {
        forkSmallKernel<<<1, SMALL_THREADS, 0, s>>>(from, to, parents, counter);
        return cudaGetLastError();
    }
    if (to.nPages > 0)
    {
        const cudaError_t err = cudaMemsetAsync(to.refs, 0, 4ll * to.nPages, s);
        if (err != cudaSuccess) return err;
    }
    forkKernel<<<blocks(std::max(n, 1ll), THREADS), THREADS, 0, s>>>(from, to, parents, counter);
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
    const int unit = unitOf(reinterpret_cast<uintptr_t>(h.pages) | reinterpret_cast<uintptr_t>(records)
                            | (unsigned long long)h.recordBytes | (unsigned long long)recordStride);
    const int perItem = itemRecords(h.recordBytes, h.pageLen), items = (h.pageLen - 1) / perItem + 1;
    if (h.nRows <= SMALL_ROWS && h.nPages <= SMALL_PAGES && h.nRows * h.recordBytes * h.pageLen <= SMALL_COPY)
    {
        appendSmallKernel<<<1, SMALL_THREADS, 0, s>>>(h, mask, w, records, recordStride, unit, perItem, items, dropped);
        return cudaGetLastError();
    }
    const cudaError_t err = cudaMemsetAsync(workspace, 0, zero, s);
    if (err != cudaSuccess) return err;
    appendShareKernel<<<blocks(h.nRows, THREADS), THREADS, 0, s>>>(h, mask, w);
    appendCountKernel<<<w.rowChunks + w.pageChunks, THREADS, 0, s>>>(h, mask, w);
    appendWriteKernel<<<blocks((long long)h.nRows * items * 32, THREADS), THREADS, 0, s>>>(h, w, records, recordStride, unit,
                                                                                          perItem, items, dropped);
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
    if (h.nPages <= SMALL_PAGES)
    {
        compactSmallKernel<<<1, SMALL_THREADS, 0, s>>>(h, w, live);
    }
    else
    {
        const cudaError_t err = cudaMemsetAsync(w.done, 0, sizeof(unsigned), s);
        if (err != cudaSuccess) return err;
        liveCountKernel<<<w.pageChunks, THREADS, 0, s>>>(h, w, live);
        compactPlanKernel<<<w.pageChunks, THREADS, 0, s>>>(h, w);
    }
    const int unit = unitOf(reinterpret_cast<uintptr_t>(h.pages) | (unsigned long long)h.recordBytes * h.pageLen);
    const int movers = std::min(h.nPages, 148 * 8);
    compactMoveKernel<<<movers + blocks((long long)h.nRows * h.rowPages, THREADS), THREADS, 0, s>>>(h, w, movers, unit);
    return cudaGetLastError();
}

void launchHistoryRead(const HistoryView& h, const long long* rows, int n, int steps, char* out, int* counts,
                       cudaStream_t s)
{
    if (n <= 0 || steps <= 0) return;
    const int unit = unitOf(reinterpret_cast<uintptr_t>(h.pages) | reinterpret_cast<uintptr_t>(out)
                            | (unsigned long long)h.recordBytes);
    const int perItem = itemRecords(h.recordBytes, std::min(32, steps)), items = (steps - 1) / perItem + 1;
    const unsigned n32 = blocks((long long)n * items * 32, THREADS);
    switch (unit)
    {
    case 16: readKernel<uint4><<<n32, THREADS, 0, s>>>(h, rows, n, steps, perItem, items, out, counts); break;
    case 8: readKernel<uint2><<<n32, THREADS, 0, s>>>(h, rows, n, steps, perItem, items, out, counts); break;
    case 4: readKernel<unsigned><<<n32, THREADS, 0, s>>>(h, rows, n, steps, perItem, items, out, counts); break;
    case 2: readKernel<unsigned short><<<n32, THREADS, 0, s>>>(h, rows, n, steps, perItem, items, out, counts); break;
    default: readKernel<uint8_t><<<n32, THREADS, 0, s>>>(h, rows, n, steps, perItem, items, out, counts); break;
    }
}

}  // namespace cb
