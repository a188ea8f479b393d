// Search operators: beam selection over a flat vocabulary and over the seven
// action heads, and the reordering of per-beam state.
//
// Beam selection.  With s_k the score of beam k and x_kv its logits, the total of
// a continuation is s_k + x_kv - log(sum of exp(x_ku) over the allowed u), and a
// step keeps the `width` largest of a group, ties to the lowest k * vocab + v.
// Within a beam the order is that of the logits, so the pass over the logits needs
// no normaliser: a warp keeps the largest of its part of a row in a sorted list
// across its lanes while it accumulates the sum.  The lists of a group's rows are
// then merged on 64-bit totals.
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

// A candidate of a row: ordered logit, complement of the action (greater is better,
// a lower action wins a tie); 0 is none.
using RowKey = u64;

// A candidate of a group: ordered 64-bit total, complement of beam * vocab + action.
struct GroupKey
{
    u64 t;
    unsigned i;
};

__device__ __forceinline__ bool better(unsigned a, unsigned b) { return a > b; }
__device__ __forceinline__ bool better(RowKey a, RowKey b) { return a > b; }
__device__ __forceinline__ bool better(const GroupKey& a, const GroupKey& b)
{
    return a.t > b.t || (a.t == b.t && a.i > b.i);
}
__device__ __forceinline__ unsigned shflXor(unsigned k, int m) { return __shfl_xor_sync(FULL, k, m); }
__device__ __forceinline__ RowKey shflXor(RowKey k, int m) { return __shfl_xor_sync(FULL, k, m); }
__device__ __forceinline__ GroupKey shflXor(const GroupKey& k, int m)
{
    return GroupKey{ __shfl_xor_sync(FULL, k.t, m), __shfl_xor_sync(FULL, k.i, m) };
}
__device__ __forceinline__ RowKey shflAt(RowKey k, int l) { return __shfl_sync(FULL, k, l); }
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

// A row of logits as a warp reads it: whole 16-byte vectors in tiles of 32 elements a
// lane, and one more element a lane for those before the first and behind the last
// vector (at most 7 each).
template <class T>
struct Row
{
    static constexpr int VE = 16 / sizeof(T);   // elements of a vector
    static constexpr int NV = 32 / VE;          // vectors of a lane per tile
    static constexpr int WORDS = 32 / Words<T>::PER;
    const T* x;
    const uint8_t* allowed;
    int head, vectors, tail, tiles, lane;
    bool wideMask;

    __device__ Row(const T* logits, const uint8_t* mask, int vocab, int l)
        : x(logits), allowed(mask), lane(l)
    {
        head = min(vocab, (int)(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T)));
        vectors = (vocab - head) / VE;
        tail = vocab - head - vectors * VE;
        tiles = (vectors + 32 * NV - 1) / (32 * NV);
        wideMask = (reinterpret_cast<uintptr_t>(mask + head) & 3) == 0;
    }
    // Element j (0 .. 31) of this lane's part of tile t, as an action.
    __device__ int action(int t, int j) const { return head + ((t * NV + j / VE) * 32 + lane) * VE + j % VE; }

    template <bool MASKED>
    __device__ __forceinline__ void load(int t, unsigned (&w)[WORDS], unsigned (&m)[8]) const
    {
        const uint4* v = reinterpret_cast<const uint4*>(x + head);
#pragma unroll
        for (int j = 0; j < NV; j++)
        {
            const int i = (t * NV + j) * 32 + lane;
            uint4 r = make_uint4(Words<T>::NONE, Words<T>::NONE, Words<T>::NONE, Words<T>::NONE);
            if (i < vectors) r = __ldcs(v + i);
            w[4 * j] = r.x;
            w[4 * j + 1] = r.y;
            w[4 * j + 2] = r.z;
            w[4 * j + 3] = r.w;
            if (MASKED)
            {
                const uint8_t* a = allowed + head + (long long)i * VE;
#pragma unroll
                for (int q = 0; q < VE / 4; q++)
                {
                    unsigned b = 0;
                    if (i < vectors)
                    {
                        if (wideMask)
                            b = __ldcs(reinterpret_cast<const unsigned*>(a + 4 * q));
                        else
                            b = a[4 * q] | a[4 * q + 1] << 8 | a[4 * q + 2] << 16 | (unsigned)a[4 * q + 3] << 24;
                    }
                    m[j * VE / 4 + q] = b;
                }
            }
        }
    }
    // What is not allowed becomes -inf.
    __device__ __forceinline__ static void hide(unsigned (&w)[WORDS], const unsigned (&m)[8])
    {
#pragma unroll
        for (int q = 0; q < 8; q++)
        {
            if (Words<T>::PER == 1)
            {
#pragma unroll
                for (int k = 0; k < 4; k++)
                    if (!(m[q] >> (8 * k) & 0xff)) w[(4 * q + k) % WORDS] = Words<T>::NONE;
            }
            else
            {
                const unsigned z = __vcmpeq4(m[q], 0);
                const unsigned lo = __byte_perm(z, 0, 0x1100), hi = __byte_perm(z, 0, 0x3322);
                w[(2 * q) % WORDS] = (w[(2 * q) % WORDS] & ~lo) | (Words<T>::NONE & lo);
                w[(2 * q + 1) % WORDS] = (w[(2 * q + 1) % WORDS] & ~hi) | (Words<T>::NONE & hi);
            }
        }
    }
    __device__ static float element(const unsigned (&w)[WORDS], int j)
    {
        return Words<T>::at(w[j / Words<T>::PER], j % Words<T>::PER);
    }
    // Largest of elements 8 k .. 8 k + 7, NaN passed over (-inf if there is nothing else).
    __device__ static float largest8(const unsigned (&w)[WORDS], int k)
    {
        constexpr int N = 8 / Words<T>::PER;
        unsigned m = w[N * k];
#pragma unroll
        for (int i = 1; i < N; i++) m = Words<T>::larger(m, w[N * k + i]);
        float f = Words<T>::at(m, 0);
        if (Words<T>::PER == 2) f = fmaxf(f, Words<T>::at(m, 1));
        return fmaxf(f, NEG_INF);
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

// The `n`-th largest (n <= 32 E) of E values a lane, as an ordered image.
template <int E>
__device__ __forceinline__ unsigned nthLargest(unsigned (&v)[E], int n, int lane)
{
    if (E == 1 && n <= 12)
    {
        // Fewer rounds of taking the maximum out than a sort has exchanges.
        unsigned mine = v[0], top = 0;
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
    sortDown(v, lane);
    unsigned r = v[0];
#pragma unroll
    for (int e = 1; e < E; e++)
        if ((n - 1) / 32 == e) r = v[e];
    return __shfl_sync(FULL, r, (n - 1) & 31);
}

// Running maximum of a row (over the warp) and, per lane, a part of the sum of
// exp(x - maximum).
struct RowSum
{
    float top = NEG_INF;
    double sum = 0.0;

    __device__ __forceinline__ float raise(float laneTop)
    {
        const float t = fromOrdered(__reduce_max_sync(FULL, ordered(laneTop)));
        if (t > top)
        {
            sum *= exp((double)top - (double)t);
            top = t;
        }
        return t;
    }
    __device__ __forceinline__ void add(float v) { sum += exp2Approx((v - (top > NEG_INF ? top : 0.f)) * LOG2E); }
    template <class T>
    __device__ __forceinline__ void add8(const unsigned (&w)[Row<T>::WORDS], int k)
    {
        const float ref = top > NEG_INF ? top : 0.f;
        float s = 0.f;
#pragma unroll
        for (int q = 0; q < 8; q++) s += exp2Approx((Row<T>::element(w, 8 * k + q) - ref) * LOG2E);
        sum += s;
    }
    // Over the warp.
    __device__ __forceinline__ void gather()
    {
#pragma unroll
        for (int m = 16; m > 0; m /= 2) sum += __shfl_xor_sync(FULL, sum, m);
    }
};

// ---- long rows: the best of each segment ----------------------------------------------

// One warp over a segment of a row: the segment's largest logits, sorted, and its sum.
//
// A tile whose maximum does not reach the list's last place costs its loads, the
// exponentials and one vote.  The first tile has no such bar yet: the width-th largest
// of the lanes' maxima is one, since at least `width` elements reach it.
template <class T, int E, bool MASKED>
__device__ __forceinline__ void scanRow(const Row<T>& row, int width, int seg, int segs, RowKey* wait,
                                        BestList<RowKey, E>& best, RowSum& sum)
{
    const int t0 = (int)((long long)row.tiles * seg / segs), t1 = (int)((long long)row.tiles * (seg + 1) / segs);
    best.init(wait, width, row.lane);
    float bar = -FLT_MAX;  // nothing below it can be kept
    bool started = false;
    unsigned next[Row<T>::WORDS], nextMask[8];
    if (t0 < t1) row.template load<MASKED>(t0, next, nextMask);
    for (int t = t0; t < t1; t++)
    {
        unsigned w[Row<T>::WORDS], m[8];
#pragma unroll
        for (int i = 0; i < Row<T>::WORDS; i++) w[i] = next[i];
        if (MASKED)
        {
#pragma unroll
            for (int i = 0; i < 8; i++) m[i] = nextMask[i];
        }
        if (t + 1 < t1) row.template load<MASKED>(t + 1, next, nextMask);
        if (MASKED) Row<T>::hide(w, m);
        float part[4];
#pragma unroll
        for (int k = 0; k < 4; k++) part[k] = Row<T>::largest8(w, k);
        const float tileTop = sum.raise(fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])));
#pragma unroll
        for (int k = 0; k < 4; k++) sum.template add8<T>(w, k);
        if (!(tileTop >= bar)) continue;
        if (!started)
        {
            started = true;
            unsigned tops[E];
#pragma unroll
            for (int e = 0; e < E; e++)
            {
                float top = part[e * (4 / E)];
#pragma unroll
                for (int k = 1; k < 4 / E; k++) top = fmaxf(top, part[e * (4 / E) + k]);
                tops[e] = top > NEG_INF ? ordered(top) : 0;
            }
            const unsigned o = nthLargest<E>(tops, width, row.lane);
            if (o) bar = fromOrdered(o);
        }
        unsigned bits = 0;
#pragma unroll
        for (int k = 0; k < 4; k++)
        {
            if (!__any_sync(FULL, part[k] >= bar)) continue;
#pragma unroll
            for (int q = 0; q < 8; q++)
                if (Row<T>::element(w, 8 * k + q) >= bar) bits |= 1u << (8 * k + q);
        }
        while (__any_sync(FULL, bits != 0))
        {
            const bool has = bits != 0;
            const int action = row.action(t, has ? __ffs(bits) - 1 : 0);
            bits &= bits - 1;
            RowKey key = 0;
            if (has) key = (RowKey)ordered(toFloat(row.x[action])) << 32 | (unsigned)~action;
            best.push(has && key > best.bar, key);
        }
        if (best.bar) bar = fmaxf(bar, fromOrdered((unsigned)(best.bar >> 32)));
    }
    if (seg == 0 && row.head + row.tail > 0)
    {
        float v;
        const int a = row.edge(v);
        sum.raise(fmaxf(v, NEG_INF));
        sum.add(v);
        const RowKey key = (RowKey)ordered(v) << 32 | (unsigned)~a;
        best.push(v >= bar && key > best.bar, key);
    }
    best.finish();
    sum.gather();
}

constexpr int ROW_WARPS = 8;
constexpr int ROW_THREADS = ROW_WARPS * 32;

// One warp per segment of a row, results to the workspace.
template <class T, int E, bool MASKED>
__global__ void __launch_bounds__(ROW_THREADS) selectRowsKernel(BeamParams p)
{
    __shared__ RowKey waitS[ROW_WARPS][32 * E + 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long item = blockIdx.x * (long long)ROW_WARPS + warp;
    if (item >= (long long)p.groups * p.beams * p.segs) return;
    const long long row = item / p.segs, g = row / p.beams;
    if (!readsLogits(p, row)) return;
    const int k = (int)(row - g * p.beams);
    BestList<RowKey, E> best;
    RowSum sum;
    scanRow<T, E, MASKED>(Row<T>(rowLogits<T>(p, g, k), rowMask(p, g, k), p.vocab, lane), p.width,
                          (int)(item - row * p.segs), p.segs, waitS[warp], best, sum);
    if (lane == 0)
    {
        p.top[item] = sum.top;
        p.sum[item] = sum.sum;
    }
#pragma unroll
    for (int e = 0; e < E; e++)
        if (e * 32 + lane < p.width) p.keys[item * p.width + e * 32 + lane] = best.list[e];
}

// ---- the best of a group -----------------------------------------------------------------

// Totals of different beams are compared through normalisers that the passes over the
// logits have to fp32 accuracy in their terms.  With u = 2^-24 and d = top - x: a term is
// off by d u (the difference), 1.25 d u (its product with log2(e), and that constant) and
// 4 u (ex2.approx); d averages at most log(vocab) <= 20.8 under the softmax; partial sums
// of eight terms add 7 u.  Together 58 u = 3.5e-6, so two totals that are further apart
// than twice that are in order.  Nearer ones are decided by normalisers in 64 bits.
constexpr double NEAR_TOTALS = 8e-6;

template <int E>
struct GroupShared
{
    GroupKey wait[ROW_WARPS][32 * E + 32];
    double red[ROW_WARPS];
    unsigned near[BEAM_MAX_BEAMS / 32];
    unsigned repair;
};

// A block orders its group's candidates and writes the group's outputs.  candidate(c,
// beam, index) gives candidate c < n: its logit, beam and beam * vocab + action (-inf for
// none); topOf(k) is the largest allowed logit of beam k; base[k] is the score minus the
// normaliser, -inf where beam k has no candidate; finished beams come on top.
template <class T, int E, class Candidate, class TopOf>
__device__ __forceinline__ void finishGroup(const BeamParams& p, long long g, int n, Candidate candidate, TopOf topOf,
                                            double* base, GroupShared<E>& sh)
{
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const long long row0 = g * p.beams;
    const int K = p.beams;
    for (int k = tid; k < BEAM_MAX_BEAMS / 32; k += ROW_THREADS) sh.near[k] = 0;
    if (tid == 0) sh.repair = 0;

    auto totalOf = [&](int c, int& beam, unsigned& index) {
        const float x = candidate(c, beam, index);
        return x > NEG_INF ? base[beam] + (double)x : (double)NEG_INF;
    };
    // Few candidates are one warp's work; more are shared out and merged pairwise.
    const int warps = n <= 256 * E ? 1 : ROW_WARPS;
    auto choose = [&]() {
        BestList<GroupKey, E> best;
        if (warp < warps)
        {
            best.init(sh.wait[warp], p.width, lane);
            for (int c0 = warp * 32; c0 < n; c0 += warps * 32)
            {
                int beam = 0;
                unsigned index = 0;
                const double total = c0 + lane < n ? totalOf(c0 + lane, beam, index) : NEG_INF;
                const GroupKey key{ ordered64(total), ~index };
                best.push(total > NEG_INF && better(key, best.bar), key);
            }
            for (int k0 = warp * 32; p.finished && k0 < K; k0 += warps * 32)
            {
                const int k = k0 + lane;
                const double total = k < K && p.finished[row0 + k] ? (double)p.scores[row0 + k] : NEG_INF;
                const GroupKey key{ ordered64(total), ~((unsigned)k * p.vocab) };
                best.push(total > NEG_INF && better(key, best.bar), key);
            }
            best.finish();
            __syncwarp();  // the buffer of waiting keys becomes the list
#pragma unroll
            for (int e = 0; e < E; e++) sh.wait[warp][e * 32 + lane] = best.list[e];
        }
        __syncthreads();
        for (int m = warps / 2; m > 0; m /= 2)
        {
            if (warp < m)
            {
                GroupKey other[E];
#pragma unroll
                for (int e = 0; e < E; e++) other[e] = sh.wait[warp + m][e * 32 + lane];
                mergeDown(best.list, other, lane);
#pragma unroll
                for (int e = 0; e < E; e++) sh.wait[warp][e * 32 + lane] = best.list[e];
            }
            __syncthreads();
        }
    };
    choose();

    // Beams whose totals are too near one another's: neighbours in the list, and what
    // lies around its last place.
    const GroupKey* list = sh.wait[0];
    const GroupKey last = list[p.width - 1];
    auto mark = [&](int beam) { atomicOr(&sh.near[beam >> 5], 1u << (beam & 31)); };
    for (int i = tid; i + 1 < p.width; i += ROW_THREADS)
    {
        const GroupKey a = list[i], b = list[i + 1];
        if (!b.t || fromOrdered64(a.t) - fromOrdered64(b.t) > NEAR_TOTALS) continue;
        const int ka = ~a.i / p.vocab, kb = ~b.i / p.vocab;
        if (ka == kb) continue;
        mark(ka);
        mark(kb);
        sh.repair = 1;
    }
    if (last.t)
    {
        const double edge = fromOrdered64(last.t);
        const int kl = ~last.i / p.vocab;
        for (int c = tid; c < n; c += ROW_THREADS)
        {
            int beam = 0;
            unsigned index = 0;
            const double total = totalOf(c, beam, index);
            if (beam == kl || !(fabs(total - edge) <= NEAR_TOTALS)) continue;
            mark(beam);
            mark(kl);
            sh.repair = 1;
        }
        for (int k = tid; p.finished && k < K; k += ROW_THREADS)
        {
            if (!p.finished[row0 + k] || k == kl || !(fabs((double)p.scores[row0 + k] - edge) <= NEAR_TOTALS)) continue;
            mark(kl);
            sh.repair = 1;
        }
    }
    __syncthreads();
    if (sh.repair)
    {
        for (int k = 0; k < K; k++)
        {
            if (!(sh.near[k >> 5] >> (k & 31) & 1) || !readsLogits(p, row0 + k)) continue;  // the same for the whole block
            const T* x = rowLogits<T>(p, g, k);
            const uint8_t* allowed = rowMask(p, g, k);
            const double t = (double)topOf(k);
            double sum = 0.0;
            for (int a = tid; a < p.vocab; a += ROW_THREADS)
                if (!allowed || allowed[a]) sum += exp((double)toFloat(x[a]) - t);
#pragma unroll
            for (int m = 16; m > 0; m /= 2) sum += __shfl_xor_sync(FULL, sum, m);
            if (lane == 0) sh.red[warp] = sum;
            __syncthreads();
            if (tid == 0)
            {
                sum = 0.0;
                for (int w = 0; w < ROW_WARPS; w++) sum += sh.red[w];
                base[k] = (double)p.scores[row0 + k] - (t + log(sum));
            }
            __syncthreads();
        }
        choose();
    }

    for (int i = tid; i < p.width; i += ROW_THREADS)
    {
        const GroupKey key = list[i];
        const unsigned index = ~key.i;
        const long long o = g * p.width + i;
        p.outScores[o] = key.t ? (float)fromOrdered64(key.t) : NEG_INF;
        p.outParents[o] = key.t ? index / p.vocab : i % K;
        p.outActions[o] = key.t ? index % p.vocab : 0;
    }
}

// From the segments' lists.
template <class T, int E>
__global__ void __launch_bounds__(ROW_THREADS) selectMergeKernel(BeamParams p)
{
    __shared__ double baseS[BEAM_MAX_BEAMS];
    __shared__ GroupShared<E> sh;
    const long long g = blockIdx.x, row0 = g * p.beams;
    const int segs = p.segs, per = segs * p.width;
    const RowKey* keys = p.keys + row0 * per;
    const float* tops = p.top + row0 * segs;
    const double* sums = p.sum + row0 * segs;
    auto topOf = [&](int k) {
        float t = NEG_INF;
        for (int s = 0; s < segs; s++) t = fmaxf(t, tops[k * segs + s]);
        return t;
    };
    for (int k = threadIdx.x; k < p.beams; k += ROW_THREADS)
    {
        double b = NEG_INF;
        const float t = readsLogits(p, row0 + k) ? topOf(k) : NEG_INF;
        if (t > NEG_INF)
        {
            double sum = 0.0;
            for (int s = 0; s < segs; s++)
            {
                // A segment without a finite logit has sum 0, or NaN where one was NaN.
                const float ts = tops[k * segs + s];
                sum += ts > NEG_INF && ts < t ? sums[k * segs + s] * exp((double)ts - (double)t) : sums[k * segs + s];
            }
            b = (double)p.scores[row0 + k] - ((double)t + log(sum));
        }
        baseS[k] = b;
    }
    __syncthreads();
    auto candidate = [&](int c, int& beam, unsigned& index) {
        beam = c / per;
        if (!(baseS[beam] > NEG_INF)) return NEG_INF;
        const RowKey key = keys[c];
        if (!key) return NEG_INF;
        index = (unsigned)beam * p.vocab + ~(unsigned)key;
        return fromOrdered((unsigned)(key >> 32));
    };
    finishGroup<T, E>(p, g, p.beams * per, candidate, topOf, baseS, sh);
}

// ---- short rows: a block per group ------------------------------------------------------

// A group's rows are read by the warps of one block.  The lanes' largest totals give a
// bar for the whole group, the width-th largest of them; the few elements that reach it
// (with a margin for rounding) are the group's candidates.  Where more reach it than
// there is room for (rows of equal logits), the rows' own best take their place.
constexpr int GROUP_MAX_BEAMS = 64;
constexpr int GROUP_MAX_KEYS = 1024;

template <class T, bool MASKED>
__global__ void __launch_bounds__(ROW_THREADS, 3) selectGroupKernel(BeamParams p)
{
    __shared__ RowKey keyS[GROUP_MAX_KEYS];        // ordered logit, beam * vocab + action
    __shared__ float topS[GROUP_MAX_BEAMS];
    __shared__ double baseS[GROUP_MAX_BEAMS];
    __shared__ unsigned laneS[ROW_THREADS];
    __shared__ float barS;
    __shared__ int countS;
    __shared__ union { RowKey wait[ROW_WARPS][64]; GroupShared<1> group; } sh;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, K = p.beams;
    const long long g = blockIdx.x;
    if (threadIdx.x == 0) countS = 0;

    unsigned w[Row<T>::WORDS], m[8];
    int held = -1, heldTile = 0;                   // the tile in registers
    float laneBest = NEG_INF;                      // largest total of the lane
    for (int k = warp; k < K; k += ROW_WARPS)
    {
        double b = NEG_INF;
        RowSum sum;
        if (readsLogits(p, g * K + k))
        {
            const Row<T> row(rowLogits<T>(p, g, k), rowMask(p, g, k), p.vocab, lane);
            float laneTop = NEG_INF;
            for (int t = 0; t < row.tiles; t++)
            {
                row.template load<MASKED>(t, w, m);
                if (MASKED) Row<T>::hide(w, m);
                held = k;
                heldTile = t;
                const float tileTop = fmaxf(fmaxf(Row<T>::largest8(w, 0), Row<T>::largest8(w, 1)),
                                            fmaxf(Row<T>::largest8(w, 2), Row<T>::largest8(w, 3)));
                laneTop = fmaxf(laneTop, tileTop);
                sum.raise(tileTop);
#pragma unroll
                for (int q = 0; q < 4; q++)
                    if ((t * Row<T>::NV + q * Row<T>::NV / 4) * 32 < row.vectors) sum.template add8<T>(w, q);
            }
            if (row.head + row.tail > 0)
            {
                float v;
                row.edge(v);
                laneTop = fmaxf(laneTop, v);
                sum.raise(fmaxf(v, NEG_INF));
                sum.add(v);
            }
            sum.gather();
            if (sum.top > NEG_INF) b = (double)p.scores[g * K + k] - ((double)sum.top + log(sum.sum));
            if (b > NEG_INF && laneTop > NEG_INF) laneBest = fmaxf(laneBest, (float)(b + (double)laneTop));
        }
        if (lane == 0)
        {
            topS[k] = sum.top;
            baseS[k] = b;
        }
    }
    laneS[threadIdx.x] = laneBest > NEG_INF ? ordered(laneBest) : 0;
    __syncthreads();
    if (warp == 0)
    {
        unsigned v[ROW_WARPS], top = 0;
#pragma unroll
        for (int i = 0; i < ROW_WARPS; i++) v[i] = laneS[i * 32 + lane];
        for (int left = p.width; left > 0;)
        {
            unsigned mine = v[0];
#pragma unroll
            for (int i = 1; i < ROW_WARPS; i++) mine = max(mine, v[i]);
            top = __reduce_max_sync(FULL, mine);
            if (top == 0) break;
            int hits = 0;
#pragma unroll
            for (int i = 0; i < ROW_WARPS; i++)
            {
                hits += v[i] == top;
                if (v[i] == top) v[i] = 0;
            }
            left -= __reduce_add_sync(FULL, hits);
        }
        if (lane == 0)
        {
            // Lower by twice NEAR_TOTALS and by eight roundings to float32.
            const float t = fromOrdered(top);
            barS = top && fabsf(t) < FLT_MAX ? t - (2.f * (float)NEAR_TOTALS + 8.f * 0x1p-24f * fabsf(t)) : NEG_INF;
        }
    }
    __syncthreads();
    const float bar = barS;
    auto offer = [&](float v, int k, int action) {
        const int at = atomicAdd(&countS, 1);
        if (at < GROUP_MAX_KEYS) keyS[at] = (RowKey)ordered(v) << 32 | ((unsigned)k * p.vocab + action);
    };
    for (int k = (K - 1 - warp) / ROW_WARPS * ROW_WARPS + warp; k >= 0 && warp < K; k -= ROW_WARPS)
    {
        const double b = baseS[k];
        if (!(b > NEG_INF)) continue;
        // Logits of this row that can reach the bar.
        const float need = b < (double)INFINITY && bar > NEG_INF ? fmaxf((float)((double)bar - b), -FLT_MAX) : -FLT_MAX;
        const float margin = need > -FLT_MAX ? need - 2.f * 0x1p-24f * fabsf(need) : need;
        if (!(topS[k] >= margin)) continue;
        const Row<T> row(rowLogits<T>(p, g, k), rowMask(p, g, k), p.vocab, lane);
        for (int t = row.tiles - 1; t >= 0; t--)
        {
            if (held != k || heldTile != t)
            {
                row.template load<MASKED>(t, w, m);
                if (MASKED) Row<T>::hide(w, m);
            }
#pragma unroll
            for (int q = 0; q < 4; q++)
            {
                if (!(Row<T>::largest8(w, q) >= margin)) continue;
#pragma unroll
                for (int i = 0; i < 8; i++)
                {
                    const float v = Row<T>::element(w, 8 * q + i);
                    if (v >= margin) offer(v, k, row.action(t, 8 * q + i));
                }
            }
        }
        if (row.head + row.tail > 0)
        {
            float v;
            const int a = row.edge(v);
            if (v >= margin) offer(v, k, a);
        }
    }
    __syncthreads();
    int n = countS;
    if (n > GROUP_MAX_KEYS)
    {
        for (int k = warp; k < K; k += ROW_WARPS)
        {
            BestList<RowKey, 1> best;
            best.init(sh.wait[warp], p.width, lane);
            RowSum sum;
            if (baseS[k] > NEG_INF)
                scanRow<T, 1, MASKED>(Row<T>(rowLogits<T>(p, g, k), rowMask(p, g, k), p.vocab, lane), p.width, 0, 1,
                                      sh.wait[warp], best, sum);
            const RowKey key = best.list[0];
            if (lane < p.width)
                keyS[k * p.width + lane] = key ? (key & ~0xffffffffull) | ((unsigned)k * p.vocab + ~(unsigned)key) : 0;
            __syncwarp();
        }
        n = K * p.width;
        __syncthreads();
    }
    auto candidate = [&](int c, int& beam, unsigned& index) {
        const RowKey key = keyS[c];
        if (!key) return NEG_INF;
        index = (unsigned)key;
        beam = index / p.vocab;
        return fromOrdered((unsigned)(key >> 32));
    };
    auto topOf = [&](int k) { return topS[k]; };
    finishGroup<T, 1>(p, g, n, candidate, topOf, baseS, sh.group);
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

__device__ __forceinline__ bool ahead(const JointKey& a, const JointKey& b) { return a.v > b.v || (a.v == b.v && a.i < b.i); }

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
            l[i] = swap ? b : a;
            l[i | s] = swap ? a : b;
        }
}

// As for the flat selection, for normalisers over seven heads: per head d averages at
// most log(3), with two additions (1.1 * 2.25 + 6) u = 8.5 u; six products; and logf's
// last place of at most 6.5, 8 u.  Together 74 u = 4.5e-6 a beam.
constexpr double NEAR_JOINT = 1e-5;

constexpr int JOINT_THREADS = 128;

// A thread per beam, the beams of a group side by side in a warp (padded to a power
// of two).  The best N joint actions of a beam are found head by head: the list of
// the best sums so far plus each choice of the next head, merged.  A choice that is
// the r-th best of its head (from 0) can only continue the first N / (r + 1) sums.
// Sums of logits are in 64 bits, so they are exact for logits within 29 binades;
// normalisers are in 32 bits first, and in 64 where two beams' totals are near.
template <class T, int N>
__global__ void __launch_bounds__(JOINT_THREADS) jointSelectKernel(BeamParams p, int lanes)
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
    const auto x = [&](int q) -> float& { return xS[q][threadIdx.x]; };  // a column of the thread's own
    const T* from = rowLogits<T>(p, reads ? g : 0, reads ? k : 0);
    const uint8_t* allowed = rowMask(p, reads ? g : 0, reads ? k : 0);
#pragma unroll
    for (int q = 0; q < ACTION_LOGITS; q++) x(q) = reads && (!allowed || allowed[q]) ? toFloat(from[q]) : NEG_INF;

    JointKey best[N];
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
                option[a] = swap ? r : l;
                option[b] = swap ? l : r;
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
                    if (ahead(c, best[N - 1 - i])) best[N - 1 - i] = c;
                }
                settle(best);
            }
        }
        if (tops > NEG_INF)
            base = (double)score - (tops + (pass == 0 ? (double)logf(product) : log(product64)));
        const bool live = reads && base > NEG_INF;
#pragma unroll
        for (int i = 0; i < N; i++)
        {
            best[i].v = live ? base + best[i].v : (double)NEG_INF;
            best[i].i += k * JOINT_ACTIONS;
        }
        if (over) best[0] = JointKey{ score > NEG_INF ? (double)score : (double)NEG_INF, k * JOINT_ACTIONS };

        // The group's: every lane of it ends with the same list.  `out` is the best that
        // another beam lost its place with.
        JointKey out{ NEG_INF, 0 };
        for (int m = 1; m < lanes; m *= 2)
        {
            JointKey other[N];
#pragma unroll
            for (int i = 0; i < N; i++)
                other[i] = JointKey{ __shfl_xor_sync(FULL, best[N - 1 - i].v, m), __shfl_xor_sync(FULL, best[N - 1 - i].i, m) };
            JointKey lost{ NEG_INF, 0 };
#pragma unroll
            for (int i = 0; i < N; i++)
            {
                const bool take = ahead(other[i], best[i]);
                const JointKey drop = take ? best[i] : other[i];
                if (take) best[i] = other[i];
                if (drop.v > lost.v) lost = drop;
            }
            settle(best);
            const JointKey theirs{ __shfl_xor_sync(FULL, out.v, m), __shfl_xor_sync(FULL, out.i, m) };
            if (theirs.v > out.v) out = theirs;
            if (lost.v > out.v) out = lost;
        }
        if (pass == 1) break;
        bool near = false;
#pragma unroll
        for (int i = 0; i < N; i++)
        {
            if (i >= p.width) continue;
            const bool edge = i + 1 >= N;
            const JointKey next = edge ? out : best[i + 1 < N ? i + 1 : i];
            near |= best[i].v - next.v <= NEAR_JOINT && next.v > NEG_INF && best[i].i / JOINT_ACTIONS != next.i / JOINT_ACTIONS;
        }
        if (!__any_sync(FULL, near)) break;
    }

    if (g >= p.groups) return;
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

// ---- state reordering --------------------------------------------------------------------

constexpr int REORDER_ARRAYS = 24;        // arrays of one launch
constexpr int REORDER_TILE = 32 * 1024;   // bytes of shared memory of a tile
constexpr int REORDER_THREADS = 256;

struct ReorderArray
{
    char* data;
    long long outerStride, inner;    // bytes
    long long firstBlock;
    int groupsPerTile, groupTiles;   // whole groups of a tile, tiles along the groups
    int units, unitTiles;            // units (of `unit` bytes) of a tile's rows, tiles along a row
    int unit;
};

struct ReorderParams
{
    ReorderArray a[REORDER_ARRAYS];
    const long long* parents;
    int count, groups, beams;
};

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
    const int rowUnits = (int)(a.inner / sizeof(U)), u0 = ut * a.units, nu = min(a.units, rowUnits - u0);
    for (int r = tid; r < rows; r += REORDER_THREADS) takenS[r] = 0;
    __syncthreads();
    for (int r = tid; r < rows; r += REORDER_THREADS)
    {
        const int j = r % K;
        const long long q = p.parents[(long long)g0 * K + r];
        const int parent = q >= 0 && q < K ? (int)q : j;  // an index outside the group leaves the slot
        parentS[r] = (short)(r - j + parent);
        if (parent != j) takenS[r - j + parent] = 1;
    }
    __syncthreads();
    U* data = reinterpret_cast<U*>(a.data + outer * a.outerStride) + (long long)g0 * K * rowUnits + u0;
    U* t = reinterpret_cast<U*>(tile);
    for (int i = tid; i < rows * nu; i += REORDER_THREADS)
    {
        const int r = i / nu, u = i - r * nu;
        if (takenS[r]) t[i] = data[(long long)r * rowUnits + u];
    }
    __syncthreads();
    for (int i = tid; i < rows * nu; i += REORDER_THREADS)
    {
        const int r = i / nu, u = i - r * nu, s = parentS[r];
        if (s != r) data[(long long)r * rowUnits + u] = t[s * nu + u];
    }
}

__global__ void __launch_bounds__(REORDER_THREADS) reorderKernel(ReorderParams p)
{
    __shared__ __align__(16) char tile[REORDER_TILE];
    __shared__ short parentS[BEAM_MAX_BEAMS];
    __shared__ uint8_t takenS[BEAM_MAX_BEAMS];
    int k = 0;
    while (k + 1 < p.count && (long long)blockIdx.x >= p.a[k + 1].firstBlock) k++;
    const ReorderArray a = p.a[k];
    switch (a.unit)
    {
    case 16: reorderTile<uint4>(p, a, tile, parentS, takenS); break;
    case 8: reorderTile<uint2>(p, a, tile, parentS, takenS); break;
    case 4: reorderTile<unsigned>(p, a, tile, parentS, takenS); break;
    case 2: reorderTile<unsigned short>(p, a, tile, parentS, takenS); break;
    default: reorderTile<uint8_t>(p, a, tile, parentS, takenS); break;
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

template <class T, int E, bool MASKED>
void launchSelect(const BeamParams& p, cudaStream_t s)
{
    const long long items = (long long)p.groups * p.beams * p.segs;
    selectRowsKernel<T, E, MASKED><<<(unsigned)((items + ROW_WARPS - 1) / ROW_WARPS), ROW_THREADS, 0, s>>>(p);
    selectMergeKernel<T, E><<<p.groups, ROW_THREADS, 0, s>>>(p);
}

template <class T, bool MASKED>
void launchSelectWidth(const BeamParams& p, cudaStream_t s)
{
    if (p.segs == 0)
        selectGroupKernel<T, MASKED><<<p.groups, ROW_THREADS, 0, s>>>(p);
    else if (p.width <= 32)
        launchSelect<T, 1, MASKED>(p, s);
    else if (p.width <= 64)
        launchSelect<T, 2, MASKED>(p, s);
    else
        launchSelect<T, 4, MASKED>(p, s);
}

template <class T>
void launchSelectMasked(const BeamParams& p, cudaStream_t s)
{
    if (p.mask)
        launchSelectWidth<T, true>(p, s);
    else
        launchSelectWidth<T, false>(p, s);
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
    const int tiles = (p.vocab + 1023) / 1024;
    // Warps the card holds at a time, at the pass's register use.
    constexpr long long WARPS = 148 * 16;
    (void)type;
    // A block per group re-reads rows of more than one tile, and its warps take the rows
    // of more than eight beams in turn.
    const bool fits = p.width <= 32 && p.width <= 16 * p.beams && p.beams <= GROUP_MAX_BEAMS
                      && p.beams * p.width <= GROUP_MAX_KEYS;
    const int turns = tiles * ((p.beams + ROW_WARPS - 1) / ROW_WARPS);
    if (fits && (turns <= 2 || (tiles <= 4 && p.groups >= 2 * 148)))
    {
        p.segs = 0;
        return 0;
    }
    p.segs = (int)std::max<long long>(1, std::min<long long>(tiles, WARPS / std::max<long long>(1, rows)));
    const long long items = rows * p.segs;
    char* c = static_cast<char*>(base);
    p.sum = reinterpret_cast<double*>(c);
    p.keys = reinterpret_cast<unsigned long long*>(c + items * 8);
    p.top = reinterpret_cast<float*>(c + items * 8 * (1 + p.width));
    return items * (8 * (1 + p.width) + 4);
}

void launchBeamSelect(const BeamParams& p, LogitType type, cudaStream_t s)
{
    if (type == LOGITS_F32)
        launchSelectMasked<float>(p, s);
    else if (type == LOGITS_BF16)
        launchSelectMasked<__nv_bfloat16>(p, s);
    else
        launchSelectMasked<__half>(p, s);
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
    for (int first = 0; first < count; first += REORDER_ARRAYS)
    {
        ReorderParams p{};
        p.parents = parents;
        p.groups = groups;
        p.beams = beams;
        long long blocks = 0;
        for (int k = first; k < count && k < first + REORDER_ARRAYS; k++)
        {
            const StateArray& in = arrays[k];
            if (in.inner == 0 || in.outer == 0) continue;
            ReorderArray& a = p.a[p.count++];
            a.data = static_cast<char*>(in.data);
            a.outerStride = in.outerStride;
            a.inner = in.inner;
            const unsigned long long bits = reinterpret_cast<uintptr_t>(in.data) | (unsigned long long)in.inner
                                            | (in.outer > 1 ? (unsigned long long)in.outerStride : 0);
            a.unit = 16;
            while (bits % a.unit) a.unit /= 2;
            const long long rowUnits = in.inner / a.unit;
            a.units = (int)std::max<long long>(1, std::min<long long>(rowUnits, REORDER_TILE / ((long long)beams * a.unit)));
            a.unitTiles = (int)((rowUnits + a.units - 1) / a.units);
            a.groupsPerTile = 1;
            if (a.unitTiles == 1)
                a.groupsPerTile = (int)std::max<long long>(1, std::min<long long>(REORDER_TILE / (beams * in.inner), BEAM_MAX_BEAMS / beams));
            a.groupTiles = (groups + a.groupsPerTile - 1) / a.groupsPerTile;
            a.firstBlock = blocks;
            blocks += in.outer * a.groupTiles * a.unitTiles;
        }
        if (blocks > 0) reorderKernel<<<(unsigned)blocks, REORDER_THREADS, 0, s>>>(p);
    }
}

void launchMoveContacts(int* contact, const long long* parents, int nSim, int beams, int nCars, cudaStream_t s)
{
    const long long n = (long long)nSim * nCars;
    moveContactsKernel<<<(unsigned)((n + REORDER_THREADS - 1) / REORDER_THREADS), REORDER_THREADS, 0, s>>>(contact, parents,
                                                                                                           nSim, beams, nCars);
}

}  // namespace cb
