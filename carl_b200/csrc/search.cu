// Search operators: beam selection over a flat vocabulary and over the seven
// action heads, and the reordering of per-beam state.
//
// Beam selection.  With s_k the score of beam k and x_kv its logits, the total of
// a continuation is s_k + x_kv - log(sum of exp(x_ku) over the allowed u), and a
// step keeps the `width` largest of a group, ties to the lowest k * vocab + v.
// The logits are read once, for the sums and for the maxima of short runs of them
// (chunks); the totals of those maxima say which few chunks can hold one of the
// best, and these are read again and ordered on 64-bit totals.
#include "search.cuh"

#include <algorithm>
#include <cfloat>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "cb_consts.cuh"

namespace cb {

namespace {

using u64 = unsigned long long;

constexpr unsigned FULL = 0xffffffffu;
constexpr float NEG_INF = -INFINITY;
constexpr float LOG2E = 1.4426950408889634f;

// ---- order-preserving integer images -------------------------------------------------

// x + 0 turns -0 into +0, which compares equal and must tie.
__device__ __forceinline__ unsigned ordered(float x)
{
    const unsigned b = __float_as_uint(x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float fromOrdered(unsigned o)
{
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ u64 ordered64(double x)
{
    const u64 b = (u64)__double_as_longlong(x + 0.0);
    return b >> 63 ? ~b : b | (1ull << 63);
}
__device__ __forceinline__ double fromOrdered64(u64 o)
{
    return __longlong_as_double((long long)(o >> 63 ? o & ~(1ull << 63) : ~o));
}

// ---- sorted lists across a warp --------------------------------------------------------

// A candidate of a group: ordered 64-bit total, complement of beam * vocab + action
// (greater is better, a lower index wins a tie); t = 0 is none.
struct GroupKey
{
    u64 t;
    unsigned i;
};

__device__ __forceinline__ bool better(const GroupKey& a, const GroupKey& b)
{
    return a.t > b.t || (a.t == b.t && a.i > b.i);
}
__device__ __forceinline__ GroupKey shflXor(const GroupKey& k, int m)
{
    return GroupKey{ __shfl_xor_sync(FULL, k.t, m), __shfl_xor_sync(FULL, k.i, m) };
}
__device__ __forceinline__ GroupKey shflAt(const GroupKey& k, int l)
{
    return GroupKey{ __shfl_sync(FULL, k.t, l), __shfl_sync(FULL, k.i, l) };
}

// Element p of a list of 32 E keys is register p / 32 of lane p % 32.  The loops over
// strides within a warp stay rolled: unrolled they made most of the library's code.
template <class Key, int E>
__device__ __forceinline__ void exchangeLanes(Key (&v)[E], int stride, int size, int lane)
{
#pragma unroll
    for (int e = 0; e < E; e++)
    {
        const bool down = ((e * 32 + lane) & size) == 0;
        const Key o = shflXor(v[e], stride);
        const bool first = (lane & stride) == 0;
        if (better(o, v[e]) == (first == down)) v[e] = o;
    }
}

template <class Key, int E>
__device__ __forceinline__ void exchangeRegisters(Key (&v)[E], int size, int lane)
{
#pragma unroll
    for (int d = E / 2; d > 0; d /= 2)
    {
        if (32 * d >= size) continue;
#pragma unroll
        for (int e = 0; e < E; e++)
        {
            if (e & d) continue;
            const bool down = ((e * 32 + lane) & size) == 0;
            const Key a = v[e], b = v[e | d];
            const bool swap = better(b, a) == down;
            v[e] = swap ? b : a;
            v[e | d] = swap ? a : b;
        }
    }
}

// Bitonic sort, largest first.
template <class Key, int E>
__device__ __forceinline__ void sortDown(Key (&v)[E], int lane)
{
#pragma unroll 1
    for (int size = 2; size <= 32 * E; size *= 2)
    {
        exchangeRegisters(v, size, lane);
#pragma unroll 1
        for (int stride = min(16, size / 2); stride > 0; stride /= 2) exchangeLanes(v, stride, size, lane);
    }
}

// The 32 E largest of two sorted lists, sorted.
template <class Key, int E>
__device__ __forceinline__ void mergeDown(Key (&list)[E], const Key (&other)[E], int lane)
{
#pragma unroll
    for (int e = 0; e < E; e++)
    {
        const Key o = shflAt(other[E - 1 - e], 31 - lane);
        if (better(o, list[e])) list[e] = o;
    }
    exchangeRegisters(list, 64 * E, lane);
#pragma unroll 1
    for (int stride = 16; stride > 0; stride /= 2) exchangeLanes(list, stride, 64 * E, lane);
}

// The best keys a warp has seen: a sorted list, and a buffer of the keys that
// passed the list's last place (`bar`) and wait to be merged.
template <class Key, int E>
struct BestList
{
    Key list[E];
    Key bar;
    Key* wait;   // 32 E + 32 keys of shared memory
    int count, last, lane;

    __device__ void init(Key* buffer, int width, int l)
    {
        wait = buffer;
        count = 0;
        last = width - 1;
        lane = l;
        bar = Key{};
#pragma unroll
        for (int e = 0; e < E; e++) list[e] = Key{};
    }
    __device__ void merge(Key (&batch)[E])
    {
        sortDown(batch, lane);
        mergeDown(list, batch, lane);
        Key b = list[0];
#pragma unroll
        for (int e = 1; e < E; e++)
            if (last / 32 == e) b = list[e];
        bar = shflAt(b, last & 31);
    }
    __device__ void push(bool pass, const Key& key)
    {
        const unsigned votes = __ballot_sync(FULL, pass);
        if (!votes) return;
        if (pass) wait[count + __popc(votes & ((1u << lane) - 1))] = key;
        count += __popc(votes);
        if (count < 32 * E) return;
        __syncwarp();
        Key batch[E];
#pragma unroll
        for (int e = 0; e < E; e++) batch[e] = wait[e * 32 + lane];
        count -= 32 * E;
        const Key rest = lane < count ? wait[32 * E + lane] : Key{};
        __syncwarp();
        if (lane < count) wait[lane] = rest;
        merge(batch);
    }
    __device__ void finish()
    {
        if (count == 0) return;
        __syncwarp();
        Key batch[E];
#pragma unroll
        for (int e = 0; e < E; e++) batch[e] = e * 32 + lane < count ? wait[e * 32 + lane] : Key{};
        count = 0;
        merge(batch);
    }
};

// ---- logits ----------------------------------------------------------------------------

__device__ __forceinline__ float toFloat(float x) { return x; }
__device__ __forceinline__ float toFloat(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float toFloat(__half x) { return __half2float(x); }

__device__ __forceinline__ float exp2Approx(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Whether a beam's logits have to be read: dead beams (score -inf or NaN) have no
// continuation, finished ones keep their score.
__device__ __forceinline__ bool readsLogits(const BeamParams& p, long long row)
{
    return p.scores[row] > NEG_INF && !(p.finished && p.finished[row]);
}
template <class T>
__device__ __forceinline__ const T* rowLogits(const BeamParams& p, long long g, int k)
{
    return static_cast<const T*>(p.logits) + g * p.groupStride + k * p.beamStride;
}
__device__ __forceinline__ const uint8_t* rowMask(const BeamParams& p, long long g, int k)
{
    return p.mask ? p.mask + g * p.maskGroupStride + k * p.maskBeamStride : nullptr;
}

// 32-bit words of logits: one float32, or two of the 16-bit types.
template <class T>
struct Words;
template <>
struct Words<float>
{
    static constexpr int PER = 1;
    static constexpr unsigned NONE = 0xff800000u;
    static __device__ __forceinline__ float at(unsigned w, int) { return __uint_as_float(w); }
    static __device__ __forceinline__ unsigned larger(unsigned a, unsigned b)
    {
        return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    }
};
template <>
struct Words<__nv_bfloat16>
{
    static constexpr int PER = 2;
    static constexpr unsigned NONE = 0xff80ff80u;
    static __device__ __forceinline__ float at(unsigned w, int q) { return __uint_as_float(q ? w & 0xffff0000u : w << 16); }
    static __device__ __forceinline__ unsigned larger(unsigned a, unsigned b)
    {
        const __nv_bfloat162 m = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
        return *reinterpret_cast<const unsigned*>(&m);
    }
};
template <>
struct Words<__half>
{
    static constexpr int PER = 2;
    static constexpr unsigned NONE = 0xfc00fc00u;
    static __device__ __forceinline__ float at(unsigned w, int q)
    {
        const __half2 h = *reinterpret_cast<__half2*>(&w);
        return q ? __high2float(h) : __low2float(h);
    }
    static __device__ __forceinline__ unsigned larger(unsigned a, unsigned b)
    {
        const __half2 m = __hmax2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
        return *reinterpret_cast<const unsigned*>(&m);
    }
};

// Sum of exp(v - ref) over eight values, two at a time (the packed fp32 instructions).
__device__ __forceinline__ u64 pack2(float a, float b)
{
    u64 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float sumExp8(const float (&v)[8], float ref)
{
    const u64 minus = pack2(-ref, -ref), scale = pack2(LOG2E, LOG2E);
    u64 total = 0;
#pragma unroll
    for (int q = 0; q < 8; q += 2)
    {
        u64 d;
        float a, b;
        asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(pack2(v[q], v[q + 1])), "l"(minus));
        asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(d), "l"(scale));
        asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(d));
        asm("add.rn.f32x2 %0, %1, %2;" : "=l"(total) : "l"(total), "l"(pack2(exp2Approx(a), exp2Approx(b))));
    }
    float a, b;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(total));
    return a + b;
}

// A row of logits as a warp reads it: 16-byte vectors, lane l those with index l mod 32,
// and one more element a lane for those before the first and behind the last vector (at
// most 7 each).  A segment is a range of vectors (a multiple of 32 but for the last); a
// lane's elements of a segment, the edges counted to the first, are a chunk.
template <class T>
struct Row
{
    static constexpr int VE = 16 / sizeof(T);   // elements of a vector
    const T* x;
    const uint8_t* allowed;
    int head, vectors, tail, lane;
    bool wideMask;

    __device__ Row(const BeamParams& p, long long g, int k, int l)
        : x(rowLogits<T>(p, g, k)), allowed(rowMask(p, g, k)), lane(l)
    {
        head = min(p.vocab, (int)(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T)));
        vectors = (p.vocab - head) / VE;
        tail = p.vocab - head - vectors * VE;
        wideMask = (reinterpret_cast<uintptr_t>(allowed + head) & 3) == 0;
    }
    // Vectors v0 + lane + 32 j below `end`; lanes beyond it read the last one, which
    // `hideBeyond` takes out again.  A j with nothing below `end` for the whole warp is left
    // out, here and by what follows.
    template <bool MASKED, int NV>
    __device__ __forceinline__ void load(int v0, int end, uint4 (&w)[NV], unsigned (&m)[NV * VE / 4]) const
    {
        const uint4* v = reinterpret_cast<const uint4*>(x + head);
#pragma unroll
        for (int j = 0; j < NV; j++)
        {
            if (v0 + 32 * j >= end) break;
            w[j] = __ldcs(v + min(v0 + 32 * j + lane, end - 1));
        }
        if (!MASKED) return;
        const uint8_t* a = allowed + head;
        if (wideMask)
        {
#pragma unroll
            for (int j = 0; j < NV; j++)
            {
                if (v0 + 32 * j >= end) break;
                const unsigned* b = reinterpret_cast<const unsigned*>(a + (long long)min(v0 + 32 * j + lane, end - 1) * VE);
#pragma unroll
                for (int q = 0; q < VE / 4; q++) m[j * VE / 4 + q] = __ldcs(b + q);
            }
        }
        else
        {
#pragma unroll
            for (int j = 0; j < NV; j++)
            {
                if (v0 + 32 * j >= end) break;
                const uint8_t* b = a + (long long)min(v0 + 32 * j + lane, end - 1) * VE;
#pragma unroll
                for (int q = 0; q < VE / 4; q++)
                    m[j * VE / 4 + q] = b[4 * q] | b[4 * q + 1] << 8 | b[4 * q + 2] << 16 | (unsigned)b[4 * q + 3] << 24;
            }
        }
    }
    __device__ __forceinline__ void hideBeyond(int v0, int end, uint4& w) const
    {
        if (v0 + 32 > end && v0 + lane >= end)
            w = make_uint4(Words<T>::NONE, Words<T>::NONE, Words<T>::NONE, Words<T>::NONE);
    }
    // What is not allowed becomes -inf.
    __device__ __forceinline__ static void hide(uint4& w, const unsigned* m)
    {
        unsigned* r = reinterpret_cast<unsigned*>(&w);
#pragma unroll
        for (int q = 0; q < VE / 4; q++)
        {
            if (VE == 4)
            {
#pragma unroll
                for (int k = 0; k < 4; k++)
                    if (!(m[q] & 0xffu << (8 * k))) r[k] = Words<T>::NONE;
            }
            else
            {
                const unsigned z = __vcmpeq4(m[q], 0);
                const unsigned lo = __byte_perm(z, 0, 0x1100), hi = __byte_perm(z, 0, 0x3322);
                r[2 * q] = (r[2 * q] & ~lo) | (Words<T>::NONE & lo);
                r[2 * q + 1] = (r[2 * q + 1] & ~hi) | (Words<T>::NONE & hi);
            }
        }
    }
    // The lane's element outside the vectors; returns its action, or -1 for none.
    __device__ int edge(float& v) const
    {
        v = NEG_INF;
        int a = -1;
        if (lane < head) a = lane;
        else if (lane >= 8 && lane < 8 + tail) a = head + vectors * VE + lane - 8;
        if (a >= 0 && (!allowed || allowed[a])) v = toFloat(x[a]);
        return a;
    }
};

// Largest of the elements of a word's worth of logits, NaN passed over.
template <class T>
__device__ __forceinline__ float largestOf(unsigned w)
{
    const float f = Words<T>::at(w, 0);
    return Words<T>::PER == 2 ? fmaxf(f, Words<T>::at(w, 1)) : f;
}

// What one pass over a segment keeps: its maximum (over the warp), the sum of
// exp(x - maximum), and every lane's largest logit.
struct Scan
{
    float top = NEG_INF, laneTop = NEG_INF;
    double sum = 0.0;

    __device__ __forceinline__ void raise(float v)
    {
        laneTop = fmaxf(laneTop, v);  // NaN is passed over: it reaches the sum alone
        const float t = fromOrdered(__reduce_max_sync(FULL, ordered(laneTop)));
        if (t > top)
        {
            if (top > NEG_INF) sum *= exp((double)top - (double)t);  // otherwise it is 0, or NaN
            top = t;
        }
    }
    __device__ __forceinline__ float ref() const { return top > NEG_INF ? top : 0.f; }
};

// One warp over vectors [begin, end) of a row, NV vectors a lane at a time.  Nothing is selected
// here: the lanes' maxima tell later which chunks can hold one of the best, and only
// those are read again.  AHEAD: the next vectors are loaded before these are used.
template <class T, bool MASKED, int NV, bool AHEAD>
__device__ __forceinline__ Scan scanRow(const Row<T>& row, int begin, int end)
{
    constexpr int VE = Row<T>::VE, MASKS = NV * VE / 4;
    Scan scan;
    uint4 w[NV], next[AHEAD ? NV : 1];
    unsigned m[MASKS], nextMask[AHEAD ? MASKS : 1];
    if constexpr (AHEAD) row.template load<MASKED, NV>(begin, end, next, nextMask);
    for (int v0 = begin; v0 < end; v0 += 32 * NV)
    {
        if constexpr (AHEAD)
        {
#pragma unroll
            for (int j = 0; j < NV; j++) w[j] = next[j];
#pragma unroll
            for (int j = 0; MASKED && j < MASKS; j++) m[j] = nextMask[j];
            row.template load<MASKED, NV>(v0 + 32 * NV, end, next, nextMask);
        }
        else
        {
            row.template load<MASKED, NV>(v0, end, w, m);
        }
        unsigned most = Words<T>::NONE;
#pragma unroll
        for (int j = 0; j < NV; j++)
        {
            if (v0 + 32 * j >= end) break;  // the same for the whole warp
            if (MASKED) Row<T>::hide(w[j], m + j * VE / 4);
            row.hideBeyond(v0 + 32 * j, end, w[j]);
            most = Words<T>::larger(most, Words<T>::larger(Words<T>::larger(w[j].x, w[j].y), Words<T>::larger(w[j].z, w[j].w)));
        }
        scan.raise(largestOf<T>(most));
        const float ref = scan.ref();
#pragma unroll
        for (int j = 0; j < NV; j += 8 / VE)
        {
            if (v0 + 32 * j >= end) break;
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; i++)
            {
                const uint4& r = w[j + i / VE];
                const int e = i % VE / Words<T>::PER;
                v[i] = Words<T>::at(e == 0 ? r.x : e == 1 ? r.y : e == 2 ? r.z : r.w, i % Words<T>::PER);
            }
            if (VE == 4 && v0 + 32 * (j + 1) >= end)
            {
#pragma unroll
                for (int i = 4; i < 8; i++) v[i] = NEG_INF;
            }
            scan.sum += sumExp8(v, ref);
        }
    }
    if (begin == 0 && row.head + row.tail > 0)
    {
        float v;
        row.edge(v);
        scan.raise(v);
        scan.sum += exp2Approx((v - scan.ref()) * LOG2E);
    }
#pragma unroll
    for (int d = 16; d > 0; d /= 2) scan.sum += __shfl_xor_sync(FULL, scan.sum, d);
    return scan;
}

constexpr int ROW_WARPS = 8;
constexpr int ROW_THREADS = ROW_WARPS * 32;

// One warp per segment of a row, results to the workspace.  Bound by memory in float32
// (64 x 16 rows of 131072: 104 us with the finishing kernel, 5.2 TB/s, where no totals are
// near); in the 16-bit types by issue (56 % of its slots) and the exponential unit at about
// eight logits a clock and SM (128 x 16 rows: 132 us, 4.1 TB/s).  Loading eight vectors at a
// time, or none ahead, measured the same.
template <class T, bool MASKED>
__global__ void __launch_bounds__(ROW_THREADS) selectRowsKernel(BeamParams p)
{
    const int lane = threadIdx.x & 31;
    const long long item = blockIdx.x * (long long)ROW_WARPS + (threadIdx.x >> 5);
    if (item >= (long long)p.groups * p.beams * p.segs) return;
    const long long r = item / p.segs, g = r / p.beams;
    if (!readsLogits(p, r)) return;
    const Row<T> row(p, g, (int)(r - g * p.beams), lane);
    const int begin = (int)(item - r * p.segs) * p.segVectors;
    const Scan scan = scanRow<T, MASKED, 4, true>(row, begin, min(row.vectors, begin + p.segVectors));
    p.chunks[item * 32 + lane] = scan.laneTop;
    if (lane == 0)
    {
        p.top[item] = scan.top;
        p.sum[item] = scan.sum;
    }
}

// ---- the best of a group -----------------------------------------------------------------

// Totals of different beams are compared through normalisers that the pass over the
// logits has to fp32 accuracy in its terms.  With u = 2^-24 and d = top - x: a term is off
// by d u (the difference), 1.25 d u (its product with log2(e), and that constant) and 4 u
// (ex2.approx); d averages at most log(vocab) <= 20.8 under the softmax; partial sums of
// eight terms add 7 u.  Together 58 u = 3.5e-6, so two totals that are further apart than
// twice that are in order.  Nearer ones are decided by normalisers in 64 bits.
constexpr double NEAR_TOTALS = 8e-6;

// Far from zero a score and a normaliser round to one of two neighbours, whatever the
// normaliser's error: totals within a few units of the last place are near as well.  (A
// total of +inf is near nothing.)
__device__ __forceinline__ double nearness(double total) { return NEAR_TOTALS + fmin(0x1p-50 * fabs(total), 1e300); }

// A continuation that reaches the group's bar.
struct Candidate
{
    double total;
    unsigned index;  // beam * vocab + action
    int beam;
};

// THREADS: a block's, or one warp's.
template <int THREADS, int E>
struct alignas(16) GroupShared
{
    static constexpr int WARPS = THREADS / 32;
    static constexpr int CHUNKS = THREADS == 32 ? 128 : 512;       // chunks that are read again
    static constexpr int CANDIDATES = THREADS == 32 ? 128 : 1024;  // and their elements that reach the bar
    GroupKey wait[WARPS][32 * E + 32];
    Candidate found[CANDIDATES];
    int chunk[CHUNKS];
    unsigned tops[THREADS];
    double red[WARPS];
    unsigned near[BEAM_MAX_BEAMS / 32];
    unsigned bar;
    int chunks, candidates, repair;
};

template <int THREADS>
__device__ __forceinline__ void groupSync()
{
    if (THREADS == 32)
        __syncwarp();
    else
        __syncthreads();
}

// A value that at least n of the threads' `mine` reach (0: there are none), nearly the
// n-th largest.
template <int THREADS, int E>
__device__ __forceinline__ unsigned nthLargest(unsigned mine, int n, int tid, GroupShared<THREADS, E>& sh)
{
    const int lane = tid & 31;
    if (THREADS > 32 || n > 12)
    {
        sh.tops[tid] = mine;
        if (tid == 0) sh.bar = 0xffffffffu;
        groupSync<THREADS>();
    }
    if (n <= 12)
    {
        // Each warp, from the largest of 32 columns: the maximum is taken out n times.
#pragma unroll
        for (int w = 0; THREADS > 32 && w < THREADS / 32; w++) mine = max(mine, sh.tops[w * 32 + lane]);
        unsigned top = 0;
        for (int left = n; left > 0;)
        {
            top = __reduce_max_sync(FULL, mine);
            const bool hit = mine == top;
            left -= __popc(__ballot_sync(FULL, hit));
            if (hit) mine = 0;
            if (top == 0) break;
        }
        return top;
    }
    // The smallest of the values with fewer than n above them.
    int above = 0;
    const uint4* t = reinterpret_cast<const uint4*>(sh.tops);
#pragma unroll 4
    for (int i = 0; i < THREADS / 4; i++)
    {
        const uint4 v = t[i];
        above += (v.x > mine) + (v.y > mine) + (v.z > mine) + (v.w > mine);
    }
    const unsigned least = __reduce_min_sync(FULL, above < n ? mine : 0xffffffffu);
    if (lane == 0) atomicMin(&sh.bar, least);
    groupSync<THREADS>();
    return sh.bar;
}

// A group's best, found and written by a block or a warp.  chunkTop(c) is the largest
// logit of chunk c = (beam * segs + segment) * 32 + lane, topOf(k) that of beam k; base[k]
// is the score minus the normaliser, -inf where beam k reads no logits or has none; and
// overOf(k) is the score of a finished beam, -inf of another.
//
// The width-th largest of the threads' largest totals is a bar that `width` elements
// reach; the chunks that reach it (lowered by the margin of the comparison) are read
// again, and their elements that do are the candidates, usually little more than
// `width`.  Each thread then counts the candidates that go before its own, which is that
// one's place.  Where there are too many for that (rows of equal logits), sorted lists
// take over, of every element if need be.
template <class T, int THREADS, int E, class ChunkTop, class TopOf, class OverOf>
__device__ __forceinline__ void finishGroup(const BeamParams& p, long long g, int tid, ChunkTop chunkTop,
                                            TopOf topOf, OverOf overOf, double* base, GroupShared<THREADS, E>& sh)
{
    using Shared = GroupShared<THREADS, E>;
    constexpr int VE = Row<T>::VE;
    const int lane = tid & 31, warp = tid >> 5;
    const long long row0 = g * p.beams;
    const int segs = THREADS == 32 ? 1 : p.segs, segVectors = THREADS == 32 ? 1 << 30 : p.segVectors;  // a warp's rows are whole
    const int K = p.beams, items = K * segs;
    const auto sync = [] { groupSync<THREADS>(); };

    if (tid == 0) sh.chunks = sh.candidates = sh.repair = 0;
    // The totals of a thread's chunks (beam k, segment s, its lane), some at a time so that
    // their loads overlap: the best, its place, and the second best.
    constexpr int AT_ONCE = THREADS == 32 ? 4 : 8;
    const int stepBeams = Shared::WARPS / segs, stepSegs = Shared::WARPS - stepBeams * segs;
    double best = NEG_INF, second = NEG_INF;
    int bestAt = 0;
    const auto eachChunk = [&](auto use) {
        int k = warp / segs, seg = warp - k * segs;
        for (int i0 = warp; i0 < items; i0 += AT_ONCE * Shared::WARPS)
        {
            float top[AT_ONCE];
            int beam[AT_ONCE];
#pragma unroll
            for (int j = 0; j < AT_ONCE; j++)
            {
                const int i = i0 + j * Shared::WARPS;
                top[j] = i < items ? chunkTop(i * 32 + lane) : NEG_INF;
                beam[j] = k;
                k += stepBeams;
                seg += stepSegs;
                if (seg >= segs)
                {
                    seg -= segs;
                    k++;
                }
            }
#pragma unroll
            for (int j = 0; j < AT_ONCE; j++)
            {
                const int i = i0 + j * Shared::WARPS;
                if (i >= items) break;
                const double b = base[beam[j]];
                // A beam that was not read has left nothing here.
                use(b > NEG_INF ? b + (double)top[j] : (double)NEG_INF, i * 32 + lane);
            }
        }
    };
    eachChunk([&](double total, int c) {
        const bool lead = total > best;
        const double less = lead ? best : total;
        if (less > second) second = less;
        if (lead)
        {
            best = total;
            bestAt = c;
        }
    });
    sync();
    // A bar that `width` elements reach, from a total of each thread that is an element's: lower
    // than the width-th largest by twice NEAR_TOTALS and by eight roundings to float32.
    const auto barOf = [&](double mine) {
        const unsigned nth = nthLargest<THREADS, E>(mine > NEG_INF ? ordered((float)mine) : 0u, p.width, tid, sh);
        const float b = nth && nth != 0xffffffffu ? fromOrdered(nth) : NEG_INF;
        return fabsf(b) < FLT_MAX ? b - (2.f * (float)NEAR_TOTALS + 8.f * 0x1p-24f * fabsf(b)) : NEG_INF;
    };
    float bar = barOf(best);

    const auto offer = [&](double total, unsigned index, int k) {
        if (!(total > NEG_INF && total >= (double)bar)) return;
        const int at = atomicAdd(&sh.candidates, 1);
        if (at < Shared::CANDIDATES) sh.found[at] = Candidate{ total, index, k };
    };
    const auto readAgain = [&](double total, int c) {
        if (!(total > NEG_INF && total >= (double)bar)) return;
        const int at = atomicAdd(&sh.chunks, 1);
        if (at < Shared::CHUNKS) sh.chunk[at] = c;
    };
    const int per = (min(segVectors, p.vocab / VE) + 31) / 32 + 1;  // vectors of a chunk, and its edge
    // The vectors of the noted chunks, shared out over the threads.
    const auto readChunks = [&](int chunks) {
        constexpr int VECTORS = THREADS == 32 ? 3 : 4;
        for (int i0 = tid; i0 < chunks * per; i0 += VECTORS * THREADS)
        {
            uint4 r[VECTORS];
            unsigned legal[VECTORS];
            int action[VECTORS], beam[VECTORS];
#pragma unroll
            for (int u = 0; u < VECTORS; u++)
            {
                const int i = i0 + u * THREADS;
                legal[u] = 0;
                if (i >= chunks * per) continue;
                const int j = i / per, v = i - j * per, c = sh.chunk[j], k = (c >> 5) / segs, seg = (c >> 5) - k * segs;
                const Row<T> row(p, g, k, c & 31);
                const int begin = THREADS == 32 ? 0 : seg * segVectors, at = begin + row.lane + 32 * v;
                beam[u] = k;
                if (v == per - 1)
                {
                    float x;
                    action[u] = begin == 0 ? row.edge(x) : -1;
                    if (action[u] >= 0) offer(base[k] + (double)x, (unsigned)k * p.vocab + action[u], k);
                }
                else if (at < row.vectors && at - begin < segVectors)
                {
                    r[u] = *(reinterpret_cast<const uint4*>(row.x + row.head) + at);
                    action[u] = row.head + at * VE;
                    legal[u] = (1u << VE) - 1;
                    if (row.allowed)
                    {
                        legal[u] = 0;
#pragma unroll
                        for (int q = 0; q < VE; q++) legal[u] |= row.allowed[action[u] + q] ? 1u << q : 0u;
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < VECTORS; u++)
            {
                if (!legal[u]) continue;
                const double b = base[beam[u]];
                // Logits that can reach the bar, then those that do.
                float need = (float)((double)bar - b);
                need = need > -FLT_MAX ? need - 2.f * 0x1p-24f * fabsf(need) : -FLT_MAX;
                const unsigned words[4] = { r[u].x, r[u].y, r[u].z, r[u].w };
                unsigned hits = 0;
#pragma unroll
                for (int q = 0; q < VE; q++)
                    if (Words<T>::at(words[q / Words<T>::PER], q % Words<T>::PER) >= need) hits |= 1u << q;
                for (hits &= legal[u]; hits; hits &= hits - 1)
                {
                    const int q = __ffs(hits) - 1, w = q / Words<T>::PER;
                    const unsigned word = w == 0 ? words[0] : w == 1 ? words[1] : w == 2 ? words[2] : words[3];
                    const float x = q % Words<T>::PER ? Words<T>::at(word, 1) : Words<T>::at(word, 0);
                    offer(b + (double)x, (unsigned)beam[u] * p.vocab + action[u] + q, beam[u]);
                }
            }
        }
    };
    // Where one beam has most of the best, its few threads' totals make a low bar and too much
    // reaches it.  What was found then, as far as there was room, gives a higher one (64 groups
    // of 64 beams over 20000, the 64 best of which are one beam's: 713 us without, 120 with).
    constexpr int ROUNDS = 6;
    bool every = false;
    int n = 0;
    for (int round = 1;; round++)
    {
        if (second > NEG_INF && second >= (double)bar)
            eachChunk(readAgain);
        else
            readAgain(best, bestAt);
        for (int k = tid; p.finished && k < K; k += THREADS) offer((double)overOf(k), (unsigned)k * p.vocab, k);
        sync();
        const int chunks = sh.chunks;
        const bool fits = chunks <= Shared::CHUNKS && (long long)chunks * per <= 1 << 30;
        if (fits) readChunks(chunks);
        sync();
        n = sh.candidates;
        if (fits && n <= THREADS) break;
        double most = NEG_INF;
        if (fits)
        {
            for (int i = tid; i < min(n, Shared::CANDIDATES); i += THREADS) most = fmax(most, sh.found[i].total);
        }
        else
        {
            for (int i = tid; i < min(chunks, Shared::CHUNKS); i += THREADS)
            {
                const int c = sh.chunk[i];
                most = fmax(most, base[(c >> 5) / segs] + (double)chunkTop(c));
            }
        }
        const float higher = barOf(most);
        if (!(higher > bar) || round == ROUNDS)
        {
            every = !fits || n > Shared::CANDIDATES;
            break;
        }
        bar = higher;
        sync();
        if (tid == 0) sh.chunks = sh.candidates = 0;
        sync();
    }
    // Marks beams whose totals are too near one another's, and computes the marked beams'
    // normalisers in 64 bits, in an order that depends on nothing but the actions.
    const auto clear = [&] {
        for (int i = tid; i < BEAM_MAX_BEAMS / 32; i += THREADS) sh.near[i] = 0;
        sync();
    };
    const auto mark = [&](int beam) {
        atomicOr(&sh.near[beam >> 5], 1u << (beam & 31));
        sh.repair = 1;
    };
    const auto marked = [&](int k) { return (sh.near[k >> 5] >> (k & 31) & 1) && readsLogits(p, row0 + k); };
    const auto repair = [&] {
        for (int k = 0; k < K; k++)
        {
            if (!marked(k)) continue;  // the same for all threads
            const T* x = rowLogits<T>(p, g, k);
            const uint8_t* allowed = rowMask(p, g, k);
            const double t = (double)topOf(k);
            double sum = 0.0;
            constexpr int AHEAD = 8;  // independent exponentials, the loads of the next ones under way
            float next[AHEAD];
            const auto load = [&](int a0) {
#pragma unroll
                for (int u = 0; u < AHEAD; u++)
                {
                    const int a = a0 + u * THREADS;
                    next[u] = a < p.vocab && (!allowed || allowed[a]) ? toFloat(x[a]) : NEG_INF;
                }
            };
            load(tid);
            for (int a0 = tid; a0 < p.vocab; a0 += AHEAD * THREADS)
            {
                double v[AHEAD];
#pragma unroll
                for (int u = 0; u < AHEAD; u++) v[u] = (double)next[u] - t;
                load(a0 + AHEAD * THREADS);
#pragma unroll
                for (int u = 0; u < AHEAD; u++) v[u] = exp(v[u]);
#pragma unroll
                for (int u = 0; u < AHEAD; u++) sum += v[u];
            }
#pragma unroll
            for (int m = 16; m > 0; m /= 2) sum += __shfl_xor_sync(FULL, sum, m);
            if (lane == 0) sh.red[warp] = sum;
            sync();
            if (tid == 0)
            {
                sum = 0.0;
                for (int w = 0; w < Shared::WARPS; w++) sum += sh.red[w];
                base[k] = (double)p.scores[row0 + k] - (t + log(sum));
            }
            sync();
        }
    };
    const auto write = [&](int place, double total, unsigned index, int beam) {
        const long long o = g * p.width + place;
        p.outScores[o] = (float)total;
        p.outParents[o] = beam;
        p.outActions[o] = index - (unsigned)beam * p.vocab;
    };
    const auto writeNone = [&](int place) {
        const long long o = g * p.width + place;
        p.outScores[o] = NEG_INF;
        p.outParents[o] = place % K;
        p.outActions[o] = 0;
    };

    if (!every && n <= THREADS)
    {
        Candidate mine{ NEG_INF, 0, -1 };
        if (tid < n) mine = sh.found[tid];
        int place = 0;
        bool near = false;
        const double range = nearness(mine.total);
#pragma unroll 4
        for (int i = 0; i < n; i++)
        {
            const Candidate c = sh.found[i];
            place += c.total > mine.total || (c.total == mine.total && c.index < mine.index);
            near |= c.beam != mine.beam && fabs(c.total - mine.total) <= range;
        }
        // Only what is near one of the first `width` places counts: the set of beams that are
        // summed again, and with it every score, depends on the totals alone and not on how
        // low the bar came to be.
        near &= tid < n && place < p.width;
        if (near) sh.repair = 1;
        sync();
        if (sh.repair)
        {
            clear();
            for (int i = 0; near && i < n; i++)
            {
                const Candidate c = sh.found[i];
                if (c.beam == mine.beam || !(fabs(c.total - mine.total) <= range)) continue;
                mark(mine.beam);
                mark(c.beam);
            }
            sync();
            repair();
            if (tid < n && marked(mine.beam))
            {
                const int action = mine.index - (unsigned)mine.beam * p.vocab;
                mine.total = base[mine.beam] + (double)toFloat(rowLogits<T>(p, g, mine.beam)[action]);
                sh.found[tid].total = mine.total;
            }
            sync();
            place = 0;
            for (int i = 0; i < n; i++)
            {
                const Candidate c = sh.found[i];
                place += c.total > mine.total || (c.total == mine.total && c.index < mine.index);
            }
        }
        if (tid < n && place < p.width) write(place, mine.total, mine.index, mine.beam);
        for (int i = n + tid; i < p.width; i += THREADS) writeNone(i);
        return;
    }

    // The elements of lane l's chunk of a segment, 32 at a time (all lanes take part; -inf is none).
    const auto eachElement = [&](const Row<T>& row, int begin, int end, int l, auto use) {
        const int elements = max(0, (end - begin - l + 31) / 32) * VE;
        for (int e0 = 0; e0 < elements; e0 += 32)
        {
            const int e = e0 + lane, action = row.head + (begin + l + e / VE * 32) * VE + e % VE;
            const bool has = e < elements && (!row.allowed || row.allowed[action]);
            use(has ? toFloat(row.x[action]) : NEG_INF, action);
        }
        float x = NEG_INF;
        const int action = begin == 0 && lane == l ? row.edge(x) : -1;
        use(x, action);
    };

    // Every element, chunk by chunk: a warp leaves out the chunks whose largest total, at
    // the lowest index it could have, would come behind its list's last place.  Rows of
    // equal logits so end after the chunks that hold their first few.
    const auto pushAll = [&](BestList<GroupKey, E>& list) {
        int k = warp / segs, seg = warp - k * segs;
        for (int i = warp; i < items; i += Shared::WARPS)
        {
            const double b = base[k];
            const Row<T> row(p, g, k, lane);
            const int begin = THREADS == 32 ? 0 : seg * segVectors, end = min(row.vectors, begin + segVectors);
            const float top = b > NEG_INF ? chunkTop(i * 32 + lane) : NEG_INF;
            const GroupKey most{ ordered64(b + (double)top),
                                 ~((unsigned)k * p.vocab + row.head + min(begin + lane, row.vectors) * VE) };
            const GroupKey edgeMost{ most.t, ~((unsigned)k * p.vocab + lane) };  // a lane in front of the vectors
            const GroupKey& bound = begin == 0 && lane < row.head ? edgeMost : most;
            unsigned left = FULL;
            while ((left &= __ballot_sync(FULL, top > NEG_INF && better(bound, list.bar))) != 0)
            {
                const int l = __ffs(left) - 1;
                left &= left - 1;
                eachElement(row, begin, end, l, [&](float x, int action) {
                    const GroupKey key{ ordered64(b + (double)x), ~((unsigned)k * p.vocab + action) };
                    list.push(x > NEG_INF && better(key, list.bar), key);
                });
            }
            k += stepBeams;
            seg += stepSegs;
            if (seg >= segs)
            {
                seg -= segs;
                k++;
            }
        }
        for (int k0 = warp * 32; p.finished && k0 < K; k0 += THREADS)
        {
            const int f = k0 + lane;
            const double total = f < K ? (double)overOf(f) : (double)NEG_INF;
            const GroupKey key{ ordered64(total), ~((unsigned)f * p.vocab) };
            list.push(total > NEG_INF && better(key, list.bar), key);
        }
    };
    const auto choose = [&]() {
        BestList<GroupKey, E> list;
        list.init(sh.wait[warp], p.width, lane);
        if (every) pushAll(list);
        for (int c0 = warp * 32; !every && c0 < n; c0 += THREADS)
        {
            GroupKey key{};
            if (c0 + lane < n) key = GroupKey{ ordered64(sh.found[c0 + lane].total), ~sh.found[c0 + lane].index };
            list.push(key.t && better(key, list.bar), key);
        }
        list.finish();
        __syncwarp();  // the buffer of waiting keys becomes the list
#pragma unroll
        for (int e = 0; e < E; e++) sh.wait[warp][e * 32 + lane] = list.list[e];
        sync();
        for (int m = Shared::WARPS / 2; m > 0; m /= 2)
        {
            if (warp < m)
            {
                GroupKey other[E];
#pragma unroll
                for (int e = 0; e < E; e++) other[e] = sh.wait[warp + m][e * 32 + lane];
                mergeDown(list.list, other, lane);
#pragma unroll
                for (int e = 0; e < E; e++) sh.wait[warp][e * 32 + lane] = list.list[e];
            }
            sync();
        }
    };
    clear();
    choose();
    const GroupKey* list = sh.wait[0];
    const GroupKey last = list[p.width - 1];
    for (int i = tid; i + 1 < p.width; i += THREADS)
    {
        const GroupKey a = list[i], b = list[i + 1];
        if (!a.t || !b.t) continue;
        const double total = fromOrdered64(a.t);
        if (!(total - fromOrdered64(b.t) <= nearness(total))) continue;
        const int ka = ~a.i / p.vocab, kb = ~b.i / p.vocab;
        if (ka == kb) continue;
        mark(ka);
        mark(kb);
    }
    const double edge = last.t ? fromOrdered64(last.t) : (double)INFINITY;
    const double edgeRange = nearness(edge);
    const int kl = ~last.i / p.vocab;
    const auto nearEdge = [&](double total, int beam) {
        if (beam == kl || !(fabs(total - edge) <= edgeRange)) return;
        mark(beam);
        mark(kl);
    };
    for (int c = tid; !every && c < n; c += THREADS) nearEdge(sh.found[c].total, sh.found[c].beam);
    if (every && last.t)
    {
        // Of the other elements those that are near the last place: largest ones of their chunks,
        // and others in the chunks whose largest is in front (fewer than `width` of them).
        if (tid == 0) sh.chunks = 0;
        sync();
        eachChunk([&](double total, int c) {
            const int k = (c >> 5) / segs;
            if (k == kl) return;
            if (fabs(total - edge) <= edgeRange)
                nearEdge(total, k);
            else if (total > edge)
                sh.chunk[atomicAdd(&sh.chunks, 1)] = c;
        });
        sync();
        for (int j = warp; j < sh.chunks; j += Shared::WARPS)
        {
            const int c = sh.chunk[j], k = (c >> 5) / segs, begin = THREADS == 32 ? 0 : ((c >> 5) - k * segs) * segVectors;
            const Row<T> row(p, g, k, lane);
            eachElement(row, begin, min(row.vectors, begin + segVectors), c & 31, [&](float x, int) {
                if (x > NEG_INF) nearEdge(base[k] + (double)x, k);
            });
        }
        for (int k = tid; p.finished && k < K; k += THREADS) nearEdge((double)overOf(k), k);
    }
    sync();
    if (sh.repair)
    {
        repair();
        for (int c = tid; !every && c < n; c += THREADS)
        {
            const Candidate f = sh.found[c];
            if (!marked(f.beam)) continue;
            const int action = f.index - (unsigned)f.beam * p.vocab;
            sh.found[c].total = base[f.beam] + (double)toFloat(rowLogits<T>(p, g, f.beam)[action]);
        }
        sync();
        choose();
    }
    for (int i = tid; i < p.width; i += THREADS)
    {
        const GroupKey key = list[i];
        if (key.t)
            write(i, fromOrdered64(key.t), ~key.i, ~key.i / p.vocab);
        else
            writeNone(i);
    }
}

// Long rows: from the segments' results.
template <class T, int E>
__global__ void __launch_bounds__(ROW_THREADS) selectMergeKernel(BeamParams p)
{
    __shared__ double baseS[BEAM_MAX_BEAMS];
    __shared__ GroupShared<ROW_THREADS, E> sh;
    const long long g = blockIdx.x, row0 = g * p.beams;
    const int segs = p.segs;
    const float* tops = p.top + row0 * segs;
    const double* sums = p.sum + row0 * segs;
    const float* chunks = p.chunks + row0 * segs * 32;
    auto topOf = [&](int k) {
        float t = NEG_INF;
        for (int s = 0; s < segs; s++) t = fmaxf(t, tops[k * segs + s]);
        return t;
    };
    // A beam's maximum and sum over its segments, by a thread where they are few, else by a
    // warp.  What a dead or finished beam left there is not looked at in the end.
    const bool alone = segs <= 4 || (segs <= 16 && p.beams > 2 * ROW_WARPS);
    const int lane = threadIdx.x & 31, lanes = alone ? 1 : 32, part = alone ? 0 : lane;
    for (int k0 = 0; k0 < p.beams; k0 += ROW_THREADS / lanes)
    {
        const int k = k0 + threadIdx.x / lanes;
        const bool on = k < p.beams;
        const float score = on ? p.scores[row0 + k] : NEG_INF;
        const bool over = on && p.finished && p.finished[row0 + k];
        float t = NEG_INF;
#pragma unroll 4
        for (int s = part; on && s < segs; s += lanes) t = fmaxf(t, tops[k * segs + s]);
        if (!alone) t = fromOrdered(__reduce_max_sync(FULL, ordered(t)));
        double sum = 0.0;
#pragma unroll 4
        for (int s = part; on && s < segs; s += lanes)
        {
            // A segment without a finite logit has sum 0, or NaN where one was NaN.
            const float ts = tops[k * segs + s];
            const double mine = sums[k * segs + s];
            sum += ts > NEG_INF && ts < t ? mine * exp((double)ts - (double)t) : mine;
        }
        if (!alone)
        {
#pragma unroll
            for (int m = 16; m > 0; m /= 2) sum += __shfl_xor_sync(FULL, sum, m);
        }
        if (on && part == 0)
            baseS[k] = score > NEG_INF && !over && t > NEG_INF ? (double)score - ((double)t + log(sum)) : (double)NEG_INF;
    }
    __syncthreads();
    finishGroup<T, ROW_THREADS, E>(
        p, g, threadIdx.x, [&](int c) { return chunks[c]; }, topOf,
        [&](int k) { return p.finished[row0 + k] ? p.scores[row0 + k] : NEG_INF; }, baseS, sh);
}

// Short rows need no workspace: what the scan of a group's rows leaves stays in shared
// memory.
constexpr int GROUP_MAX_BEAMS = 32;
constexpr int GROUP_MAX_WIDTH = 16;
constexpr int GROUP_WARPS = 8;   // warps of a group's block

// What the scan of a group's rows leaves, in shared memory.
struct GroupRows
{
    double *base, *sum;                 // [beams]
    float *top, *score, *over, *chunk;  // [beams] (over: a finished beam's score), [beams, 32]

    __host__ __device__ static int bytes(int beams) { return (beams * 156 + 15) / 16 * 16; }
    __device__ GroupRows(char* m, int beams)
        : base(reinterpret_cast<double*>(m)), sum(base + beams), top(reinterpret_cast<float*>(sum + beams)),
          score(top + beams), over(score + beams), chunk(over + beams)
    {
    }
};

// The rows of a group from beam k0 on, every `step`-th.
template <class T, bool MASKED>
__device__ __forceinline__ void scanGroup(const BeamParams& p, long long g, int k0, int step, int lane, GroupRows& r)
{
    for (int k = k0; k < p.beams; k += step)
    {
        const float score = p.scores[g * p.beams + k];
        const bool over = p.finished && p.finished[g * p.beams + k];
        Scan scan;
        if (score > NEG_INF && !over)
        {
            const Row<T> row(p, g, k, lane);
            scan = scanRow<T, MASKED, 8, false>(row, 0, row.vectors);
        }
        r.chunk[k * 32 + lane] = scan.laneTop;
        if (lane == 0)
        {
            r.top[k] = scan.top;
            r.sum[k] = scan.sum;
            r.score[k] = score;
            r.over[k] = over ? score : NEG_INF;
        }
    }
}

template <class T>
__device__ __forceinline__ void finishRows(const BeamParams& p, long long g, int lane, GroupRows& r, GroupShared<32, 1>& sh)
{
    if (lane < p.beams)
        r.base[lane] = r.top[lane] > NEG_INF ? (double)r.score[lane] - ((double)r.top[lane] + log(r.sum[lane]))
                                             : (double)NEG_INF;
    __syncwarp();
    finishGroup<T, 32, 1>(
        p, g, lane, [&](int c) { return r.chunk[c]; }, [&](int k) { return r.top[k]; }, [&](int k) { return r.over[k]; },
        r.base, sh);
}

// A block reads a group's rows, its first warp finishes.  Bound by latency: 4096 groups of 8
// beams over 648 with a mask take 45 us, their 18.8 M instructions 17 us of issue and the
// bytes 14.  A warp waits for its next row's score, then for the row, and 26 % of the warps'
// places are taken.
template <class T, bool MASKED>
__global__ void __launch_bounds__(GROUP_WARPS * 32, 3) selectGroupKernel(BeamParams p)
{
    extern __shared__ __align__(16) char groupMem[];
    __shared__ GroupShared<32, 1> sh;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    GroupRows r(groupMem, p.beams);
    scanGroup<T, MASKED>(p, blockIdx.x, warp, blockDim.x >> 5, lane, r);
    __syncthreads();
    if (warp == 0) finishRows<T>(p, blockIdx.x, lane, r, sh);
}

// ---- selection over the action heads ---------------------------------------------------

constexpr int HEADS = 7;
constexpr int JOINT_ACTIONS = 3 * 3 * 3 * 2 * 2 * 3 * 2;
__host__ __device__ constexpr int headSize(int h) { return h < 3 || h == 5 ? 3 : 2; }

struct JointKey
{
    double v;  // sum of logits, then total; -inf: none
    int i;     // action, then beam * JOINT_ACTIONS + action
};

// Without branches, as the exchanges below.
__device__ __forceinline__ bool ahead(const JointKey& a, const JointKey& b)
{
    return (bool)((a.v > b.v) | ((a.v == b.v) & (a.i < b.i)));
}
__device__ __forceinline__ JointKey pick(bool first, const JointKey& a, const JointKey& b)
{
    return JointKey{ first ? a.v : b.v, first ? a.i : b.i };
}

// Sorts a bitonic list, best first.
template <int N>
__device__ __forceinline__ void settle(JointKey (&l)[N])
{
#pragma unroll
    for (int s = N / 2; s > 0; s /= 2)
#pragma unroll
        for (int i = 0; i < N; i++)
        {
            if (i & s) continue;
            const JointKey a = l[i], b = l[i | s];
            const bool swap = ahead(b, a);
            l[i] = pick(swap, b, a);
            l[i | s] = pick(swap, a, b);
        }
}

// A logit's last bit, in binades below its first.
template <class T>
__device__ constexpr int lastBit();
template <>
__device__ constexpr int lastBit<float>() { return 23; }
template <>
__device__ constexpr int lastBit<__nv_bfloat16>() { return 7; }
template <>
__device__ constexpr int lastBit<__half>() { return 10; }

// The best of a beam's totals, one after another; the first of equal ones stays in front.
// The six choices of the last two heads side by side: 24576 groups of 8 such beams take 154
// us (36 if they were not looked through; an action at a time took 399), and 70 where five of
// them have one (41 without: the time of the warp that comes last).
template <class X, int N>
__device__ __forceinline__ void bestTotals(const X& x, double base, JointKey (&best)[N])
{
#pragma unroll
    for (int i = 0; i < N; i++) best[i] = JointKey{ NEG_INF, 0 };
    double low[3], last[2];
#pragma unroll
    for (int q = 0; q < 3; q++) low[q] = (double)x(13 + q);
#pragma unroll
    for (int q = 0; q < 2; q++) last[q] = (double)x(16 + q);
#pragma unroll 1
    for (int a = 0; a < JOINT_ACTIONS / 6; a++)
    {
        const int a2 = a >> 2, a1 = a2 / 3, a0 = a1 / 3;
        const double sum = (double)x(a0) + (double)x(3 + a1 - 3 * a0) + (double)x(6 + a2 - 3 * a1) + (double)x(9 + (a >> 1 & 1))
                           + (double)x(11 + (a & 1));
        double total[6];
        bool any = false;
#pragma unroll
        for (int q = 0; q < 6; q++)
        {
            // -inf (an action not allowed) and NaN (that, and a base of +inf) go before nothing.
            total[q] = base + (sum + low[q / 2] + last[q % 2]);
            any |= total[q] > best[N - 1].v;
        }
        if (!any) continue;
#pragma unroll 1
        for (int q = 0; q < 6; q++)
        {
            const double v = q == 0 ? total[0] : q == 1 ? total[1] : q == 2 ? total[2] : q == 3 ? total[3] : q == 4 ? total[4] : total[5];
            const JointKey key{ v, 6 * a + q };
            if (!(v > best[N - 1].v)) continue;
#pragma unroll
            for (int i = N - 1; i > 0; i--) best[i] = v > best[i - 1].v ? best[i - 1] : v > best[i].v ? key : best[i];
            if (v > best[0].v) best[0] = key;
        }
    }
}

// As for the flat selection, for normalisers over seven heads: per head d averages at
// most log(3), with two additions (1.1 * 2.25 + 6) u = 8.5 u; six products; and logf's
// last place of at most 6.5, 8 u.  Together 74 u = 4.5e-6 a beam.
constexpr double NEAR_JOINT = 1e-5;

constexpr int JOINT_THREADS = 128;
// Blocks that an SM has to hold (0: no limit).  Lists of 8 take 72 registers and 43.1 us with
// the limit, 80 and 44.0 without (24576 groups of 8 beams; one group 8.2 and 9.4); of 16, 96 and
// 93, 128 and 107 (12288 of 16).  For lists of 32 a limit of two blocks costs 312 us, none 248
// (6144 of 32), and for lists of 4 one of nine 24.5, none 25.2, but 19.7 against 19.0 where a
// group is one beam.
constexpr int jointBlocks(int n) { return n == 8 ? 7 : n == 16 ? 5 : 0; }

// 196608 rows of 18 logits in 24576 groups: 43 us.  25.5 M instructions are 22 us of issue
// and the bytes 4; the rest is waiting for the 64-bit pipe and for loads with a third of the
// warps' places taken, and the few warps that take the 64-bit pass.  Blocks of 64 threads
// measured the same, a limit of 48 registers 3 us more, outputs through shared memory 7.
//
// A thread per beam, the beams of a group side by side in a warp (padded to a power
// of two).  The best N joint actions of a beam are found head by head: the list of
// the best sums so far plus each choice of the next head, merged.  A choice that is
// the r-th best of its head (from 0) can only continue the first N / (r + 1) sums.
// Sums of logits are in 64 bits; normalisers are in 32 bits first, and in 64 where two
// beams' totals are near.
//
// Lists of sums are in the order of the totals, equal ones by their action, where sums that
// differ make totals that do.  A logit is a whole multiple of its last bit's value, and so
// is a sum of the last bit q of the smallest logit (2^-23 of its binade, in the 16-bit types
// 2^-10 and 2^-7).  While the sums and the base stay below 2^52 q, sums are exact, differ by
// q at least and are apart by a unit in the last place of any total.  A beam beyond that (a
// float32 logit 29 binades below the total, or a score of +inf) has its 648 totals looked
// through in turn, in the second pass.
template <class T, int N>
__global__ void __launch_bounds__(JOINT_THREADS, jointBlocks(N)) jointSelectKernel(BeamParams p, int lanes)
{
    const int lane = threadIdx.x & 31, K = p.beams;
    const long long warp = (blockIdx.x * (long long)JOINT_THREADS + threadIdx.x) >> 5;
    const long long g = warp * (32 / lanes) + lane / lanes;
    const int k = lane % lanes;
    const bool on = g < p.groups && k < K;
    const long long row = g * K + k;
    const float score = on ? p.scores[row] : NEG_INF;
    const bool over = on && p.finished && p.finished[row];
    const bool reads = on && !over && score > NEG_INF;
    __shared__ float xS[ACTION_LOGITS][JOINT_THREADS];
    __shared__ double ownS[N][JOINT_THREADS];
    const auto x = [&](int q) -> float& { return xS[q][threadIdx.x]; };  // a column of the thread's own
    const auto own = [&](int i) -> double& { return ownS[i][threadIdx.x]; };
    const T* from = rowLogits<T>(p, reads ? g : 0, reads ? k : 0);
    const uint8_t* allowed = rowMask(p, reads ? g : 0, reads ? k : 0);
    unsigned least = 0xffffffffu;  // image of the smallest logit's size, less one (0 wraps)
    float most = 0.f;              // largest logit's size
#pragma unroll
    for (int q = 0; q < ACTION_LOGITS; q++)
    {
        const float v = reads && (!allowed || allowed[q]) ? toFloat(from[q]) : NEG_INF;
        least = min(least, (__float_as_uint(v) & 0x7fffffffu) - 1);
        most = fmaxf(most, v > NEG_INF ? fabsf(v) : 0.f);
        x(q) = v;
    }

    JointKey best[N];
    bool again = false, anyAgain = false;  // the group's second pass, and the warp's
    for (int pass = 0; pass < 2; pass++)
    {
        // The normaliser (NaN or +inf among the logits makes it NaN, an empty head -inf),
        // and the beam's best joint actions.
        double tops = 0.0, base = NEG_INF;
        float product = 1.f;
        double product64 = 1.0;
#pragma unroll
        for (int i = 0; i < N; i++) best[i] = JointKey{ NEG_INF, 0 };
        best[0].v = 0.0;
        int at = 0;
#pragma unroll 1
        for (int h = 0; h < HEADS; h++)
        {
            const int size = headSize(h);
            const float v[3] = { x(at), x(at + 1), size == 3 ? x(at + 2) : NEG_INF };
            at += size;
            const float top = fmaxf(fmaxf(v[0], v[1]), v[2]);
            tops += (double)top;
            if (pass == 0)
            {
                float sum = 0.f;
#pragma unroll
                for (int q = 0; q < 3; q++) sum += exp2Approx((v[q] - top) * LOG2E);
                product *= sum;
            }
            else
            {
                double sum = 0.0;
#pragma unroll 1
                for (int q = 0; q < 3; q++) sum += exp((double)(q == 0 ? v[0] : q == 1 ? v[1] : v[2]) - (double)top);
                product64 *= sum;
            }
            // The head's choices, best first.
            JointKey option[3];
#pragma unroll
            for (int q = 0; q < 3; q++) option[q] = JointKey{ (double)v[q], q };
            auto order = [&](int a, int b) {
                const JointKey l = option[a], r = option[b];
                const bool swap = ahead(r, l);
                option[a] = pick(swap, r, l);
                option[b] = pick(swap, l, r);
            };
            order(0, 1);
            order(1, 2);
            order(0, 1);
            JointKey before[N];
#pragma unroll
            for (int i = 0; i < N; i++)
            {
                before[i] = best[i];
                best[i] = JointKey{ before[i].v + option[0].v, before[i].i * size + option[0].i };
            }
#pragma unroll
            for (int r = 1; r < 3; r++)
            {
                if (r >= size) continue;
#pragma unroll
                for (int i = 0; i < N / (r + 1); i++)
                {
                    const JointKey c{ before[i].v + option[r].v, before[i].i * size + option[r].i };
                    best[N - 1 - i] = pick(ahead(c, best[N - 1 - i]), c, best[N - 1 - i]);
                }
                settle(best);
            }
        }
        if (tops > NEG_INF)
            base = (double)score - (tops + (pass == 0 ? (double)logf(product) : log(product64)));
        const bool live = reads && base > NEG_INF;
        // 2^52 q, the exponent's field of q being that of the smallest logit less its bits.
        const double limit = __longlong_as_double((long long)(max((int)(least >> 23), 1) - 75 - lastBit<T>() + 1023) << 52);
        const bool merges = live && !(fabs(base) + 7.0 * (double)most < limit);
        if (pass == 1 && merges) bestTotals(x, base, best);
#pragma unroll
        for (int i = 0; i < N; i++)
        {
            if (pass == 0 || !merges) best[i].v = live ? base + best[i].v : (double)NEG_INF;
            best[i].i += k * JOINT_ACTIONS;
        }
        if (over) best[0] = JointKey{ score > NEG_INF ? (double)score : (double)NEG_INF, k * JOINT_ACTIONS };

        // The group's: every lane of it ends with the same list.  A beam's own totals stay in
        // shared memory, to tell what it has left behind the last place.
        if (pass == 0)
        {
#pragma unroll
            for (int i = 0; i < N; i++) own(i) = best[i].v;
        }
        for (int m = 1; m < lanes; m *= 2)
        {
            JointKey other[N];
#pragma unroll
            for (int i = 0; i < N; i++)
                other[i] = JointKey{ __shfl_xor_sync(FULL, best[N - 1 - i].v, m), __shfl_xor_sync(FULL, best[N - 1 - i].i, m) };
#pragma unroll
            for (int i = 0; i < N; i++) best[i] = pick(ahead(other[i], best[i]), other[i], best[i]);
            settle(best);
        }
        // Two kept places in a row of different beams, or the last one and the best that another
        // beam has left, may be in the wrong order if they are near.  Any other two of different
        // beams that are near have such a pair between them.
        if (pass == 0)
        {
            bool near = false;
            int kept = 0;  // of this beam
            JointKey last = best[0];
#pragma unroll
            for (int i = 0; i < N; i++)
            {
                if (i >= p.width) continue;
                if (i > 0)
                    near |= last.v - best[i].v <= NEAR_JOINT + 0x1p-50 * fabs(last.v) && best[i].v > NEG_INF
                            && last.i / JOINT_ACTIONS != best[i].i / JOINT_ACTIONS;
                last = best[i];
                kept += last.i / JOINT_ACTIONS == k;
            }
            const double left = kept < N ? own(kept) : (double)NEG_INF;
            near |= last.v - left <= NEAR_JOINT + 0x1p-50 * fabs(last.v) && left > NEG_INF && last.i / JOINT_ACTIONS != k;
            near |= merges && kept > 0;  // the values of such a list are right, their actions may not be
            const unsigned votes = __ballot_sync(FULL, near), group = (lanes < 32 ? (1u << lanes) - 1 : FULL) << (lane - k);
            again = votes & group;
            anyAgain = votes != 0;
        }
        // A group's result does not depend on whether others beside it need the second pass.
        if (g < p.groups && again == (pass == 1))
        {
#pragma unroll
            for (int i = 0; i < N; i++)
            {
                if (i >= p.width || (i & (lanes - 1)) != k) continue;
                const bool some = best[i].v > NEG_INF;
                const long long o = g * p.width + i;
                const int beam = best[i].i / JOINT_ACTIONS;
                p.outScores[o] = (float)best[i].v;
                p.outParents[o] = some ? beam : i % K;
                int rest = some ? best[i].i - beam * JOINT_ACTIONS : 0;
#pragma unroll
                for (int h = HEADS - 1; h >= 0; h--)
                {
                    p.outActions[o * HEADS + h] = rest % headSize(h);
                    rest /= headSize(h);
                }
            }
        }
        if (!anyAgain) break;
    }
}

// ---- state reordering --------------------------------------------------------------------
//
// Every byte of a moved row is read and written once; the kernels differ in how a block
// finds them.  The word-major state of 32768 sims of 3v3, whose 24-byte rows fill every
// 32-byte sector, is 188 MB of sectors in 36 us (77 us row by row in the largest unit): 5.3
// TB/s at the L2 cache, of which 129 MB reach memory (3.9 TB/s).  It waits for loads and at
// the barrier of a slab.  Rows of whole 16-byte columns go through registers (reorderRowsKernel: 32768 sims'
// observations, hidden states and actions, 53.6 us of bytes at the copy rate, in 73);
// short rows, as the simulator's words of a few cars, through shared memory as one dense
// run of whole groups (reorderRunsKernel); anything else, and what is too small for more
// than one launch to pay, in the row's largest unit (reorderTilesKernel).

constexpr int REORDER_ARRAYS = 24;        // arrays of one launch
constexpr int REORDER_TILE = 32 * 1024;   // bytes of shared memory of a tile
constexpr int REORDER_THREADS = 256;

struct ReorderArray
{
    char* data;
    long long outer, outerStride, inner;  // slabs; bytes
    long long firstBlock;
    int groupsPerTile, groupTiles;        // whole groups of a tile, tiles along the groups
    int units, unitTiles;                 // units (of `unit` bytes) of a tile's rows, tiles along a row
    int unit;
};

struct ReorderParams
{
    ReorderArray a[REORDER_ARRAYS];
    const long long* parents;
    int count, groups, beams;
};

// The slot's parent; an index outside the group leaves the slot.
__device__ __forceinline__ int parentOf(const ReorderParams& p, long long row, int slot)
{
    const long long q = p.parents[row];
    return q >= 0 && q < p.beams ? (int)q : slot;
}

__device__ __forceinline__ const ReorderArray& arrayOf(const ReorderParams& p)
{
    int k = 0;
    while (k + 1 < p.count && (long long)blockIdx.x >= p.a[k + 1].firstBlock) k++;
    return p.a[k];
}

// A tile is whole groups by a range of columns: the rows that some slot takes are
// read into shared memory, then the slots that change are written.
template <class U>
__device__ void reorderTile(const ReorderParams& p, const ReorderArray& a, char* tile, short* parentS, uint8_t* takenS)
{
    const int tid = threadIdx.x, K = p.beams;
    long long b = blockIdx.x - a.firstBlock;
    const int ut = (int)(b % a.unitTiles);
    b /= a.unitTiles;
    const int gt = (int)(b % a.groupTiles);
    const long long outer = b / a.groupTiles;
    const int g0 = gt * a.groupsPerTile, ng = min(a.groupsPerTile, p.groups - g0), rows = ng * K;
    const long long rowUnits = a.inner / (long long)sizeof(U), u0 = (long long)ut * a.units;
    const int nu = (int)min((long long)a.units, rowUnits - u0);
    for (int r = tid; r < rows; r += REORDER_THREADS) takenS[r] = 0;
    __syncthreads();
    for (int r = tid; r < rows; r += REORDER_THREADS)
    {
        const int j = r % K, parent = parentOf(p, (long long)g0 * K + r, j);
        parentS[r] = (short)(r - j + parent);
        if (parent != j) takenS[r - j + parent] = 1;
    }
    __syncthreads();
    U* data = reinterpret_cast<U*>(a.data + outer * a.outerStride) + (long long)g0 * K * rowUnits + u0;
    U* t = reinterpret_cast<U*>(tile);
    for (int i = tid; i < rows * nu; i += REORDER_THREADS)
    {
        const int r = i / nu, u = i - r * nu;
        if (takenS[r]) t[i] = data[r * rowUnits + u];
    }
    __syncthreads();
    for (int i = tid; i < rows * nu; i += REORDER_THREADS)
    {
        const int r = i / nu, u = i - r * nu, s = parentS[r];
        if (s != r) data[r * rowUnits + u] = t[s * nu + u];
    }
}

__global__ void __launch_bounds__(REORDER_THREADS) reorderTilesKernel(ReorderParams p)
{
    __shared__ __align__(16) char tile[REORDER_TILE];
    __shared__ short parentS[BEAM_MAX_BEAMS];
    __shared__ uint8_t takenS[BEAM_MAX_BEAMS];
    const ReorderArray a = arrayOf(p);
    switch (a.unit)
    {
    case 16: reorderTile<uint4>(p, a, tile, parentS, takenS); break;
    case 8: reorderTile<uint2>(p, a, tile, parentS, takenS); break;
    case 4: reorderTile<unsigned>(p, a, tile, parentS, takenS); break;
    case 2: reorderTile<unsigned short>(p, a, tile, parentS, takenS); break;
    default: reorderTile<uint8_t>(p, a, tile, parentS, takenS); break;
    }
}

// Short rows of whole words: a tile is a dense run of whole groups, read and written in
// 16-byte vectors, permuted by words in shared memory.  The words' places are worked out
// once and used for several slabs; the next slab is loaded while this one is permuted.
constexpr int RUN_VECTORS = 2;                                         // of a thread
constexpr int RUN_WORDS = REORDER_THREADS * RUN_VECTORS * 4;           // of a tile
constexpr int RUN_SLABS = 8;                                           // of a block

__global__ void __launch_bounds__(REORDER_THREADS) reorderRunsKernel(ReorderParams p)
{
    __shared__ __align__(16) unsigned tile[2][RUN_WORDS];
    short* parentS = reinterpret_cast<short*>(tile[1]);  // until the first slab is permuted
    const ReorderArray a = arrayOf(p);
    const int tid = threadIdx.x, K = p.beams, W = (int)(a.inner / 4);
    const long long b = blockIdx.x - a.firstBlock;
    const int gt = (int)(b % a.groupTiles);
    const long long s0 = b / a.groupTiles * RUN_SLABS, s1 = min(a.outer, s0 + RUN_SLABS);
    const int g0 = gt * a.groupsPerTile, ng = min(a.groupsPerTile, p.groups - g0), rows = ng * K, words = rows * W;
    char* data = a.data + (long long)g0 * K * a.inner;

    uint4 next[RUN_VECTORS];
    const auto load = [&](long long s) {
        const uint4* from = reinterpret_cast<const uint4*>(data + s * a.outerStride);
#pragma unroll
        for (int u = 0; u < RUN_VECTORS; u++)
            if ((tid + u * REORDER_THREADS) * 4 + 3 < words) next[u] = from[tid + u * REORDER_THREADS];
    };
    load(s0);
    for (int r = tid; r < rows; r += REORDER_THREADS)
    {
        const int j = r % K;
        parentS[r] = (short)(r - j + parentOf(p, (long long)g0 * K + r, j));
    }
    __syncthreads();
    short source[RUN_VECTORS][4];
    bool moves[RUN_VECTORS];
#pragma unroll
    for (int u = 0; u < RUN_VECTORS; u++)
    {
        moves[u] = false;
#pragma unroll
        for (int q = 0; q < 4; q++)
        {
            const int w = (tid + u * REORDER_THREADS) * 4 + q, r = w / W;
            source[u][q] = (short)(w < words ? parentS[r] * W + (w - r * W) : 0);
            moves[u] |= w < words && source[u][q] != w;
        }
    }
    // The words behind the last whole vector, fewer than four.
    const int tail = words & ~3, tw = tail + tid;
    const bool hasTail = tw < words;
    const int tailSource = hasTail ? parentS[tw / W] * W + tw % W : 0;
    for (long long s = s0, turn = 0; s < s1; s++, turn ^= 1)
    {
        unsigned* t = tile[turn];
        unsigned* slab = reinterpret_cast<unsigned*>(data + s * a.outerStride);
#pragma unroll
        for (int u = 0; u < RUN_VECTORS; u++)
            if ((tid + u * REORDER_THREADS) * 4 + 3 < words) reinterpret_cast<uint4*>(t)[tid + u * REORDER_THREADS] = next[u];
        if (hasTail) t[tw] = slab[tw];
        __syncthreads();
        if (s + 1 < s1) load(s + 1);
#pragma unroll
        for (int u = 0; u < RUN_VECTORS; u++)
        {
            const int v = tid + u * REORDER_THREADS;
            if (!moves[u] || v * 4 + 3 >= words) continue;
            reinterpret_cast<uint4*>(slab)[v] = make_uint4(t[source[u][0]], t[source[u][1]], t[source[u][2]], t[source[u][3]]);
        }
        if (hasTail) slab[tw] = t[tailSource];
    }
}

// Rows of whole 16-byte columns: a thread holds its column of a group's rows.
constexpr int COLUMN_BEAMS = 16;
constexpr int COLUMN_THREADS = 128;

template <int BEAMS>
__global__ void __launch_bounds__(COLUMN_THREADS) reorderRowsKernel(ReorderParams p)
{
    __shared__ int parentS[BEAMS];
    __shared__ unsigned takenS;
    const ReorderArray a = arrayOf(p);
    const int tid = threadIdx.x, K = p.beams;
    const long long b = blockIdx.x - a.firstBlock, og = b / a.unitTiles, outer = og / p.groups, g = og - outer * p.groups;
    const long long columns = a.inner / 16, c0 = (b - og * a.unitTiles) * a.units, c1 = min(columns, c0 + a.units);
    if (tid == 0) takenS = 0;
    __syncthreads();
    if (tid < K)
    {
        const int parent = parentOf(p, g * K + tid, tid);
        parentS[tid] = parent;
        if (parent != tid) atomicOr(&takenS, 1u << parent);
    }
    __syncthreads();
    const unsigned taken = takenS;
    if (!taken) return;
    uint4* data = reinterpret_cast<uint4*>(a.data + outer * a.outerStride + g * K * a.inner);
    for (long long c = c0 + tid; c < c1; c += COLUMN_THREADS)
    {
        uint4 held[BEAMS];
#pragma unroll
        for (int k = 0; k < BEAMS; k++)
            if (taken >> k & 1) held[k] = data[k * columns + c];
#pragma unroll
        for (int k = 0; k < BEAMS; k++)
        {
            if (!(taken >> k & 1)) continue;
            for (int j = 0; j < K; j++)  // the same for the whole block
                if (parentS[j] == k && j != k) data[j * columns + c] = held[k];
        }
    }
}

__global__ void __launch_bounds__(REORDER_THREADS) moveContactsKernel(int* contact, const long long* parents, int nSim,
                                                                      int beams, int nCars)
{
    const long long car = blockIdx.x * (long long)REORDER_THREADS + threadIdx.x;
    if (car >= (long long)nSim * nCars) return;
    const int sim = (int)(car / nCars), j = sim % beams;
    const long long parent = parents[sim];
    if (parent < 0 || parent >= beams || parent == j) return;
    if (contact[car] >= 0) contact[car] += (j - (int)parent) * nCars;
}

template <class T>
void launchSelect(const BeamParams& p, cudaStream_t s)
{
    if (p.segs == 0)
    {
        const int bytes = GroupRows::bytes(p.beams);
        // About 16 warps to an SM: fewer warps to a group waste less in its serial part, more
        // shorten a lone group (8 beams over 648 with a mask, us with 1 / 2 / 4 / 8 warps: 148
        // groups 16 / 11 / 8.6 / 7.5; 1184: 20 / 15 / 19 / 21; 16384: 123 / 144 / 145 / 207).
        int warps = GROUP_WARPS;
        while (warps > 1 && (long long)p.groups * warps > 148 * 24) warps /= 2;
        const int threads = std::min(warps, p.beams) * 32;
        if (p.mask)
            selectGroupKernel<T, true><<<p.groups, threads, bytes, s>>>(p);
        else
            selectGroupKernel<T, false><<<p.groups, threads, bytes, s>>>(p);
        return;
    }
    const long long items = (long long)p.groups * p.beams * p.segs;
    const unsigned blocks = (unsigned)((items + ROW_WARPS - 1) / ROW_WARPS);
    if (p.mask)
        selectRowsKernel<T, true><<<blocks, ROW_THREADS, 0, s>>>(p);
    else
        selectRowsKernel<T, false><<<blocks, ROW_THREADS, 0, s>>>(p);
    if (p.width <= 32)
        selectMergeKernel<T, 1><<<p.groups, ROW_THREADS, 0, s>>>(p);
    else if (p.width <= 64)
        selectMergeKernel<T, 2><<<p.groups, ROW_THREADS, 0, s>>>(p);
    else
        selectMergeKernel<T, 4><<<p.groups, ROW_THREADS, 0, s>>>(p);
}

template <class T, int N>
void launchJoint(const BeamParams& p, cudaStream_t s)
{
    int lanes = 1;
    while (lanes < p.beams) lanes *= 2;
    const long long threads = ((long long)p.groups * lanes + 31) / 32 * 32;
    jointSelectKernel<T, N><<<(unsigned)((threads + JOINT_THREADS - 1) / JOINT_THREADS), JOINT_THREADS, 0, s>>>(p, lanes);
}

template <class T>
void launchJointWidth(const BeamParams& p, cudaStream_t s)
{
    if (p.width <= 4)
        launchJoint<T, 4>(p, s);
    else if (p.width <= 8)
        launchJoint<T, 8>(p, s);
    else if (p.width <= 16)
        launchJoint<T, 16>(p, s);
    else
        launchJoint<T, 32>(p, s);
}

}  // namespace

long long planBeamSelect(BeamParams& p, LogitType type, void* base)
{
    const long long rows = (long long)p.groups * p.beams;
    const int tiles = (int)(((long long)p.vocab * (type == LOGITS_F32 ? 4 : 2) + 2047) / 2048);  // of a warp's pass
    // Short rows are one block's work per group.
    const int turns = tiles * ((p.beams + ROW_WARPS - 1) / ROW_WARPS);
    if (p.width <= GROUP_MAX_WIDTH && p.beams <= GROUP_MAX_BEAMS && (turns <= 4 || (tiles <= 16 && p.groups >= 4 * 148)))
    {
        p.segs = 0;
        return 0;
    }
    // Warps the card holds at a time, at the pass's register use.
    constexpr long long WARPS = 148 * 32;
    // At least four tiles to a segment, and at most 256 segments to a group: more of them cost
    // the block that finishes it more than they save the readers (4 groups of 32 beams over
    // 131072 in bf16: 42 us without this bound, 33 with 512, 27 with 256, 37 with 128).
    const long long most = std::min<long long>((tiles + 3) / 4, std::max(1, 256 / p.beams));
    p.segs = (int)std::max<long long>(1, std::min<long long>(most, WARPS / std::max<long long>(1, rows)));
    const int perVector = type == LOGITS_F32 ? 4 : 8, blocks = (p.vocab / perVector + 31) / 32;
    p.segVectors = std::max(1, (blocks + p.segs - 1) / p.segs) * 32;
    const long long items = rows * p.segs;
    char* c = static_cast<char*>(base);
    p.sum = reinterpret_cast<double*>(c);
    p.top = reinterpret_cast<float*>(c + items * 8);
    p.chunks = reinterpret_cast<float*>(c + items * 12);
    return items * (12 + 128);
}

void launchBeamSelect(const BeamParams& p, LogitType type, cudaStream_t s)
{
    if (type == LOGITS_F32)
        launchSelect<float>(p, s);
    else if (type == LOGITS_BF16)
        launchSelect<__nv_bfloat16>(p, s);
    else
        launchSelect<__half>(p, s);
}

void launchJointSelect(const BeamParams& p, LogitType type, cudaStream_t s)
{
    if (type == LOGITS_F32)
        launchJointWidth<float>(p, s);
    else if (type == LOGITS_BF16)
        launchJointWidth<__nv_bfloat16>(p, s);
    else
        launchJointWidth<__half>(p, s);
}

void launchReorder(const StateArray* arrays, int count, const long long* parents, int groups, int beams, cudaStream_t s)
{
    enum Form { TILES, RUNS, ROWS, FORMS };
    constexpr long long MOST_BLOCKS = 0x7fffffff;
    ReorderParams p[FORMS] = {};
    long long blocks[FORMS] = {};
    const auto flush = [&](int f) {
        if (blocks[f] > 0)
        {
            const unsigned n = (unsigned)blocks[f];
            if (f == TILES)
                reorderTilesKernel<<<n, REORDER_THREADS, 0, s>>>(p[f]);
            else if (f == RUNS)
                reorderRunsKernel<<<n, REORDER_THREADS, 0, s>>>(p[f]);
            else if (beams <= 8)
                reorderRowsKernel<8><<<n, COLUMN_THREADS, 0, s>>>(p[f]);
            else
                reorderRowsKernel<COLUMN_BEAMS><<<n, COLUMN_THREADS, 0, s>>>(p[f]);
        }
        p[f].count = 0;
        blocks[f] = 0;
    };
    const long long rows = (long long)groups * beams;
    long long bytes = 0;
    for (int k = 0; k < count; k++) bytes += rows * arrays[k].outer * arrays[k].inner;
    // Below this a second launch costs more than the better form saves.
    const bool small = bytes < (1 << 20);
    for (int k = 0; k < count; k++)
    {
        const StateArray& in = arrays[k];
        if (in.inner == 0 || in.outer == 0) continue;
        ReorderArray a{};
        a.outerStride = in.outerStride;
        a.inner = in.inner;
        const unsigned long long base = reinterpret_cast<uintptr_t>(in.data) | (in.outer > 1 ? (unsigned long long)in.outerStride : 0);
        const unsigned long long bits = base | (unsigned long long)in.inner;
        int form = TILES;
        long long slabs = 1, perSlabs = 0;  // blocks of so many slabs
        if (!small && bits % 16 == 0 && in.inner >= 256 && beams <= COLUMN_BEAMS)
        {
            form = ROWS;
            a.units = 4 * COLUMN_THREADS;
            a.unitTiles = (int)((in.inner / 16 + a.units - 1) / a.units);
            perSlabs = (long long)groups * a.unitTiles;
        }
        else if (!small && base % 16 == 0 && in.inner % 4 == 0 && in.inner / 4 * beams <= RUN_WORDS / 4)
        {
            form = RUNS;
            const int words = (int)(in.inner / 4) * beams;
            a.groupsPerTile = RUN_WORDS / words / 4 * 4;  // tiles start at whole vectors
            a.groupTiles = (int)(((long long)groups + a.groupsPerTile - 1) / a.groupsPerTile);
            slabs = RUN_SLABS;
            perSlabs = a.groupTiles;
        }
        else
        {
            a.unit = 16;
            while (bits % a.unit) a.unit /= 2;
            const long long rowUnits = in.inner / a.unit;
            a.units = (int)std::max<long long>(1, std::min<long long>(rowUnits, REORDER_TILE / ((long long)beams * a.unit)));
            a.unitTiles = (int)((rowUnits + a.units - 1) / a.units);
            a.groupsPerTile = 1;
            if (a.unitTiles == 1)
                a.groupsPerTile = (int)std::max<long long>(
                    1, std::min<long long>(REORDER_TILE / (beams * in.inner), BEAM_MAX_BEAMS / beams));
            a.groupTiles = (int)(((long long)groups + a.groupsPerTile - 1) / a.groupsPerTile);
            perSlabs = (long long)a.groupTiles * a.unitTiles;
        }
        // A launch takes MOST_BLOCKS; an array of more (many small slabs) is split at its slabs.
        const long long most = std::max(1ll, MOST_BLOCKS / perSlabs) * slabs;
        ReorderParams& q = p[form];
        for (long long s0 = 0; s0 < in.outer; s0 += most)
        {
            a.data = static_cast<char*>(in.data) + s0 * in.outerStride;
            a.outer = std::min(most, in.outer - s0);
            const long long n = (a.outer + slabs - 1) / slabs * perSlabs;
            if (q.count == REORDER_ARRAYS || blocks[form] + n > MOST_BLOCKS) flush(form);
            q.parents = parents;
            q.groups = groups;
            q.beams = beams;
            a.firstBlock = blocks[form];
            q.a[q.count++] = a;
            blocks[form] += n;
        }
    }
    for (int f = 0; f < FORMS; f++) flush(f);
}

void launchMoveContacts(int* contact, const long long* parents, int nSim, int beams, int nCars, cudaStream_t s)
{
    const long long n = (long long)nSim * nCars;
    moveContactsKernel<<<(unsigned)((n + REORDER_THREADS - 1) / REORDER_THREADS), REORDER_THREADS, 0, s>>>(contact, parents,
                                                                                                           nSim, beams, nCars);
}

}  // namespace cb
