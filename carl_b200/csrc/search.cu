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

__device__ __forceinline__ bool better(RowKey a, RowKey b) { return a > b; }
__device__ __forceinline__ bool better(const GroupKey& a, const GroupKey& b)
{
    return a.t > b.t || (a.t == b.t && a.i > b.i);
}
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

// Element p of a list of 32 E keys is register p / 32 of lane p % 32.
template <class Key, int E>
__device__ __forceinline__ void exchange(Key (&v)[E], int stride, int size, int lane)
{
    if (stride >= 32)
    {
        const int d = stride / 32;
#pragma unroll
        for (int e = 0; e < E; e++)
        {
            if (e & d) continue;
            const bool down = ((e * 32 + lane) & size) == 0;
            const Key a = v[e], b = v[(e | d) < E ? (e | d) : e];
            const bool ok = better(b, a) != down;
            v[e] = ok ? a : b;
            v[(e | d) < E ? (e | d) : e] = ok ? b : a;
        }
    }
    else
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
}

// Bitonic sort, largest first.
template <class Key, int E>
__device__ __forceinline__ void sortDown(Key (&v)[E], int lane)
{
#pragma unroll
    for (int size = 2; size <= 32 * E; size *= 2)
#pragma unroll
        for (int stride = size / 2; stride > 0; stride /= 2) exchange(v, stride, size, lane);
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
#pragma unroll
    for (int stride = 16 * E; stride > 0; stride /= 2) exchange(list, stride, 64 * E, lane);
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

__device__ __forceinline__ void unpack(const uint4& r, float (&v)[4], float)
{
    v[0] = __uint_as_float(r.x);
    v[1] = __uint_as_float(r.y);
    v[2] = __uint_as_float(r.z);
    v[3] = __uint_as_float(r.w);
}
__device__ __forceinline__ void unpack(const uint4& r, float (&v)[8], __nv_bfloat16)
{
    const unsigned w[4] = { r.x, r.y, r.z, r.w };
#pragma unroll
    for (int k = 0; k < 4; k++)
    {
        v[2 * k] = __uint_as_float(w[k] << 16);
        v[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
    }
}
__device__ __forceinline__ void unpack(const uint4& r, float (&v)[8], __half)
{
    const unsigned w[4] = { r.x, r.y, r.z, r.w };
#pragma unroll
    for (int k = 0; k < 4; k++)
    {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
        v[2 * k] = f.x;
        v[2 * k + 1] = f.y;
    }
}

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

// ---- the pass over the logits --------------------------------------------------------

constexpr int ROW_WARPS = 8;

// One warp per segment of a row: the segment's largest logits, their maximum and
// the sum of exp(x - maximum).
template <class T, int E, bool MASKED>
__global__ void __launch_bounds__(ROW_WARPS * 32) selectRowsKernel(BeamParams p)
{
    constexpr int VE = 16 / sizeof(T);  // elements of a 16-byte load
    constexpr int NV = 32 / VE;         // loads of a lane per tile of 1024 elements
    __shared__ RowKey waitS[ROW_WARPS][32 * E + 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long item = blockIdx.x * (long long)ROW_WARPS + warp;
    if (item >= (long long)p.groups * p.beams * p.segs) return;
    const long long row = item / p.segs;
    const int seg = (int)(item - row * p.segs);
    if (!readsLogits(p, row)) return;
    const long long g = row / p.beams, k = row - g * p.beams;
    const T* x = static_cast<const T*>(p.logits) + g * p.groupStride + k * p.beamStride;
    const uint8_t* allowed = MASKED ? p.mask + g * p.maskGroupStride + k * p.maskBeamStride : nullptr;

    const int head = min(p.vocab, (int)(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T)));
    const int vectors = (p.vocab - head) / VE, tail = p.vocab - head - vectors * VE;
    const int tiles = (vectors + 32 * NV - 1) / (32 * NV);
    const int t0 = (int)((long long)tiles * seg / p.segs), t1 = (int)((long long)tiles * (seg + 1) / p.segs);
    const bool wideMask = MASKED && (reinterpret_cast<uintptr_t>(allowed + head) % VE) == 0;

    BestList<RowKey, E> best;
    best.init(waitS[warp], p.width, lane);
    float top = NEG_INF;
    double sum = 0.0;

    auto absorb = [&](float laneTop) {
        if (laneTop != laneTop) laneTop = NEG_INF;  // NaN reaches the sum, not the maximum
        const unsigned o = __reduce_max_sync(FULL, ordered(laneTop));
        const float t = fromOrdered(o);
        if (t > top)
        {
            sum *= exp((double)top - (double)t);
            top = t;
        }
    };
    auto offer = [&](float v, int action) {
        const float bar = best.bar ? fromOrdered((unsigned)(best.bar >> 32)) : NEG_INF;
        const RowKey key = ((RowKey)ordered(v) << 32) | (unsigned)~action;
        best.push(v >= bar && v > NEG_INF && key > best.bar, key);
    };

    // The elements before the first and behind the last whole vector.
    if (seg == 0 && head + tail > 0)
    {
        const bool front = lane < head, back = lane >= 8 && lane < 8 + tail;
        const int a = front ? lane : head + vectors * VE + lane - 8;
        float v = NEG_INF;
        if ((front || back) && (!MASKED || allowed[a])) v = toFloat(x[a]);
        absorb(v);
        sum += exp2Approx((v - (top > NEG_INF ? top : 0.f)) * LOG2E);
        offer(v, a);
    }
    const uint4* xv = reinterpret_cast<const uint4*>(x + head);
    for (int t = t0; t < t1; t++)
    {
        float v[32];
        uint4 raw[NV];
#pragma unroll
        for (int j = 0; j < NV; j++)
        {
            const int i = (t * NV + j) * 32 + lane;
            if (i < vectors) raw[j] = __ldcs(xv + i);
        }
#pragma unroll
        for (int j = 0; j < NV; j++)
        {
            const int i = (t * NV + j) * 32 + lane;
            float f[VE];
            unpack(raw[j], f, T());
            bool ok[VE];
#pragma unroll
            for (int q = 0; q < VE; q++) ok[q] = i < vectors;
            if (MASKED && i < vectors)
            {
                const uint8_t* m = allowed + head + i * VE;
                if (wideMask)
                {
                    unsigned w[2];
                    w[0] = __ldcs(reinterpret_cast<const unsigned*>(m));
                    if (VE == 8) w[1] = __ldcs(reinterpret_cast<const unsigned*>(m) + 1);
#pragma unroll
                    for (int q = 0; q < VE; q++) ok[q] = (w[q / 4] >> (8 * (q & 3)) & 0xffu) != 0;
                }
                else
                {
#pragma unroll
                    for (int q = 0; q < VE; q++) ok[q] = m[q] != 0;
                }
            }
#pragma unroll
            for (int q = 0; q < VE; q++) v[j * VE + q] = ok[q] ? f[q] : NEG_INF;
        }
        float laneTop = v[0];
#pragma unroll
        for (int j = 1; j < 32; j++) laneTop = fmaxf(laneTop, v[j]);
        absorb(laneTop);
        const float ref = top > NEG_INF ? top : 0.f;
#pragma unroll
        for (int j = 0; j < 32; j += 8)
        {
            float s = 0.f;
#pragma unroll
            for (int q = 0; q < 8; q++) s += exp2Approx((v[j + q] - ref) * LOG2E);
            sum += s;
        }
        const float bar = best.bar ? fromOrdered((unsigned)(best.bar >> 32)) : NEG_INF;
        if (__any_sync(FULL, laneTop >= bar && laneTop > NEG_INF))
        {
#pragma unroll
            for (int j = 0; j < 32; j++) offer(v[j], head + ((t * NV + j / VE) * 32 + lane) * VE + j % VE);
        }
    }
    best.finish();
#pragma unroll
    for (int m = 16; m > 0; m /= 2) sum += __shfl_xor_sync(FULL, sum, m);
    if (lane == 0)
    {
        p.top[item] = top;
        p.sum[item] = sum;
    }
#pragma unroll
    for (int e = 0; e < E; e++)
        if (e * 32 + lane < p.width) p.keys[item * p.width + e * 32 + lane] = best.list[e];
}

// ---- the merge of a group --------------------------------------------------------------

constexpr int MERGE_WARPS = 8;
constexpr int MERGE_THREADS = MERGE_WARPS * 32;

// Totals of different beams are compared through normalisers that the pass above
// has to fp32 accuracy in its terms.  Its error in the logarithm of a sum: per term
// the rounding of x - top and of its product with log2(e) (2^-24 each, and 2^-26 for
// the constant) times |x - top|, whose mean under the softmax is at most
// log(vocab) <= 21.5; ex2.approx's 2^-22; seven additions of 2^-24.  Together below
// 3.5e-6, so two totals that are further apart than twice that are in order.  Nearer
// ones are decided by normalisers in 64 bits.
constexpr double NEAR_TOTALS = 8e-6;

// Sorted best of the block's warps in listS[0] (all threads return after it is there).
template <int E>
__device__ void mergeWarps(BestList<GroupKey, E>& best, GroupKey (*listS)[32 * E + 32], int warp, int lane)
{
    __syncthreads();  // the buffers of waiting keys become the lists
#pragma unroll
    for (int e = 0; e < E; e++) listS[warp][e * 32 + lane] = best.list[e];
    __syncthreads();
    for (int n = MERGE_WARPS / 2; n > 0; n /= 2)
    {
        if (warp < n)
        {
            GroupKey other[E];
#pragma unroll
            for (int e = 0; e < E; e++) other[e] = listS[warp + n][e * 32 + lane];
            mergeDown(best.list, other, lane);
#pragma unroll
            for (int e = 0; e < E; e++) listS[warp][e * 32 + lane] = best.list[e];
        }
        __syncthreads();
    }
}

template <class T, int E>
__global__ void __launch_bounds__(MERGE_THREADS) selectMergeKernel(BeamParams p)
{
    __shared__ double baseS[BEAM_MAX_BEAMS];   // score minus normaliser; -inf: no candidate among the lists
    __shared__ GroupKey waitS[MERGE_WARPS][32 * E + 32];
    __shared__ unsigned nearS[BEAM_MAX_BEAMS / 32];
    __shared__ double redS[MERGE_WARPS];
    __shared__ unsigned repairS;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const long long g = blockIdx.x, row0 = g * p.beams;
    const int K = p.beams, per = p.segs * p.width;

    for (int k = tid; k < K; k += MERGE_THREADS)
    {
        double base = NEG_INF;
        if (readsLogits(p, row0 + k))
        {
            const float* top = p.top + (row0 + k) * p.segs;
            const double* sum = p.sum + (row0 + k) * p.segs;
            float t = NEG_INF;
            for (int s = 0; s < p.segs; s++) t = fmaxf(t, top[s]);
            double n = 0.0;
            if (t > NEG_INF)
            {
                for (int s = 0; s < p.segs; s++)
                {
                    // A segment without a finite logit has sum 0, or NaN where one was NaN.
                    n += top[s] > NEG_INF ? sum[s] * exp((double)top[s] - (double)t) : sum[s];
                }
                base = (double)p.scores[row0 + k] - ((double)t + log(n));
            }
        }
        baseS[k] = base;
    }
    for (int k = tid; k < BEAM_MAX_BEAMS / 32; k += MERGE_THREADS) nearS[k] = 0;
    if (tid == 0) repairS = 0;
    __syncthreads();

    auto totalOf = [&](long long c, int& beam, unsigned& index) {
        beam = (int)(c / per);
        const double base = baseS[beam];
        if (!(base > NEG_INF)) return (double)NEG_INF;
        const RowKey key = p.keys[row0 * per + c];
        if (!key) return (double)NEG_INF;
        index = (unsigned)beam * p.vocab + ~(unsigned)key;
        return base + (double)fromOrdered((unsigned)(key >> 32));
    };
    const long long n = (long long)K * per;
    BestList<GroupKey, E> best;
    auto choose = [&]() {
        best.init(waitS[warp], p.width, lane);
        for (long long c0 = warp * 32; c0 < n; c0 += MERGE_THREADS)
        {
            const long long c = c0 + lane;
            int beam = 0;
            unsigned index = 0;
            const double total = c < n ? totalOf(c, beam, index) : NEG_INF;
            const GroupKey key{ ordered64(total), ~index };
            best.push(total > NEG_INF && better(key, best.bar), key);
        }
        for (int k0 = warp * 32; p.finished && k0 < K; k0 += MERGE_THREADS)
        {
            const int k = k0 + lane;
            const double total = k < K && p.finished[row0 + k] ? (double)p.scores[row0 + k] : NEG_INF;
            const GroupKey key{ ordered64(total), ~((unsigned)k * p.vocab) };
            best.push(total > NEG_INF && better(key, best.bar), key);
        }
        best.finish();
        mergeWarps(best, waitS, warp, lane);
    };
    choose();

    // Beams whose totals are too near one another's: neighbours in the list, and what
    // lies around its last place.
    const GroupKey last = waitS[0][p.width - 1];
    auto mark = [&](int beam) { atomicOr(&nearS[beam >> 5], 1u << (beam & 31)); };
    for (int i = tid; i + 1 < p.width; i += MERGE_THREADS)
    {
        const GroupKey a = waitS[0][i], b = waitS[0][i + 1];
        if (!b.t || fromOrdered64(a.t) - fromOrdered64(b.t) > NEAR_TOTALS) continue;
        const int ka = ~a.i / p.vocab, kb = ~b.i / p.vocab;
        if (ka == kb) continue;
        mark(ka);
        mark(kb);
        repairS = 1;
    }
    if (last.t)
    {
        const double edge = fromOrdered64(last.t);
        const int kl = ~last.i / p.vocab;
        for (long long c = tid; c < n; c += MERGE_THREADS)
        {
            int beam;
            unsigned index;
            const double total = totalOf(c, beam, index);
            if (beam == kl || !(fabs(total - edge) <= NEAR_TOTALS)) continue;
            mark(beam);
            mark(kl);
            repairS = 1;
        }
        for (int k = tid; p.finished && k < K; k += MERGE_THREADS)
        {
            if (!p.finished[row0 + k] || k == kl || !(fabs((double)p.scores[row0 + k] - edge) <= NEAR_TOTALS)) continue;
            mark(kl);
            repairS = 1;
        }
    }
    __syncthreads();
    if (repairS)
    {
        for (int k = 0; k < K; k++)
        {
            if (!(nearS[k >> 5] >> (k & 31) & 1) || !readsLogits(p, row0 + k)) continue;  // the same for the whole block
            const T* x = static_cast<const T*>(p.logits) + g * p.groupStride + k * p.beamStride;
            const uint8_t* allowed = p.mask ? p.mask + g * p.maskGroupStride + k * p.maskBeamStride : nullptr;
            float t = NEG_INF;
            for (int s = 0; s < p.segs; s++) t = fmaxf(t, p.top[(row0 + k) * p.segs + s]);
            double sum = 0.0;
            for (int a = tid; a < p.vocab; a += MERGE_THREADS)
                if (!allowed || allowed[a]) sum += exp((double)toFloat(x[a]) - (double)t);
#pragma unroll
            for (int m = 16; m > 0; m /= 2) sum += __shfl_xor_sync(FULL, sum, m);
            if (lane == 0) redS[warp] = sum;
            __syncthreads();
            if (tid == 0)
            {
                sum = 0.0;
                for (int w = 0; w < MERGE_WARPS; w++) sum += redS[w];
                baseS[k] = (double)p.scores[row0 + k] - ((double)t + log(sum));
            }
            __syncthreads();
        }
        choose();
    }

    for (int i = tid; i < p.width; i += MERGE_THREADS)
    {
        const GroupKey key = waitS[0][i];
        const unsigned index = ~key.i;
        const long long o = g * p.width + i;
        p.outScores[o] = key.t ? (float)fromOrdered64(key.t) : NEG_INF;
        p.outParents[o] = key.t ? index / p.vocab : i % K;
        p.outActions[o] = key.t ? index % p.vocab : 0;
    }
}

// ---- selection over the action heads ---------------------------------------------------

constexpr int HEADS = 7;
constexpr int JOINT_ACTIONS = 3 * 3 * 3 * 2 * 2 * 3 * 2;
__host__ __device__ constexpr int headSize(int h) { return h < 3 || h == 5 ? 3 : 2; }

// One block per group.  The continuations of a beam are the 648 sums of one logit
// per head; sums and normalisers are in 64 bits.
template <class T>
__global__ void __launch_bounds__(MERGE_THREADS) jointSelectKernel(BeamParams p)
{
    __shared__ double baseS[JOINT_MAX_BEAMS];
    __shared__ double logitS[JOINT_MAX_BEAMS][ACTION_LOGITS];
    __shared__ GroupKey waitS[MERGE_WARPS][64];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const long long g = blockIdx.x, row0 = g * p.beams;
    const int K = p.beams;
    for (int k = tid; k < K; k += MERGE_THREADS)
    {
        double base = NEG_INF;
        if (readsLogits(p, row0 + k))
        {
            const T* x = static_cast<const T*>(p.logits) + g * p.groupStride + k * p.beamStride;
            const uint8_t* allowed = p.mask ? p.mask + g * p.maskGroupStride + k * p.maskBeamStride : nullptr;
            double norm = 0.0;
            int at = 0;
            for (int h = 0; h < HEADS; h++)
            {
                double top = NEG_INF, sum = 0.0;
                for (int q = 0; q < headSize(h); q++)
                {
                    const double v = !allowed || allowed[at + q] ? (double)toFloat(x[at + q]) : NEG_INF;
                    logitS[k][at + q] = v;
                    top = v > top ? v : top;
                }
                for (int q = 0; q < headSize(h); q++)
                {
                    const double v = logitS[k][at + q];
                    sum += exp(v - (top > NEG_INF ? top : 0.0));
                }
                norm += (top > NEG_INF ? top : 0.0) + log(sum);
                at += headSize(h);
            }
            base = (double)p.scores[row0 + k] - norm;
        }
        baseS[k] = base;
    }
    __syncthreads();
    BestList<GroupKey, 1> best;
    best.init(waitS[warp], p.width, lane);
    for (int c0 = warp * 32; c0 < K * JOINT_ACTIONS; c0 += MERGE_THREADS)
    {
        const int c = c0 + lane, beam = c / JOINT_ACTIONS;
        double total = NEG_INF;
        if (c < K * JOINT_ACTIONS && baseS[beam] > NEG_INF)
        {
            int rest = c - beam * JOINT_ACTIONS, at = ACTION_LOGITS;
            double sum = 0.0;
            for (int h = HEADS - 1; h >= 0; h--)
            {
                at -= headSize(h);
                sum += logitS[beam][at + rest % headSize(h)];
                rest /= headSize(h);
            }
            total = baseS[beam] + sum;
        }
        const GroupKey key{ ordered64(total), ~(unsigned)c };
        best.push(total > NEG_INF && better(key, best.bar), key);
    }
    if (p.finished && warp == 0)
    {
        const double total = lane < K && p.finished[row0 + lane] ? (double)p.scores[row0 + lane] : NEG_INF;
        const GroupKey key{ ordered64(total), ~(unsigned)(lane * JOINT_ACTIONS) };
        best.push(total > NEG_INF && better(key, best.bar), key);
    }
    best.finish();
    mergeWarps(best, waitS, warp, lane);
    for (int i = tid; i < p.width; i += MERGE_THREADS)
    {
        const GroupKey key = waitS[0][i];
        const unsigned index = ~key.i;
        const long long o = g * p.width + i;
        p.outScores[o] = key.t ? (float)fromOrdered64(key.t) : NEG_INF;
        p.outParents[o] = key.t ? index / JOINT_ACTIONS : i % K;
        int rest = key.t ? index % JOINT_ACTIONS : 0;
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

template <class T, int E>
void launchSelect(const BeamParams& p, cudaStream_t s)
{
    const long long items = (long long)p.groups * p.beams * p.segs;
    const unsigned blocks = (unsigned)((items + ROW_WARPS - 1) / ROW_WARPS);
    if (p.mask)
        selectRowsKernel<T, E, true><<<blocks, ROW_WARPS * 32, 0, s>>>(p);
    else
        selectRowsKernel<T, E, false><<<blocks, ROW_WARPS * 32, 0, s>>>(p);
    selectMergeKernel<T, E><<<p.groups, MERGE_THREADS, 0, s>>>(p);
}

template <class T>
void launchSelectWidth(const BeamParams& p, cudaStream_t s)
{
    if (p.width <= 32)
        launchSelect<T, 1>(p, s);
    else if (p.width <= 64)
        launchSelect<T, 2>(p, s);
    else
        launchSelect<T, 4>(p, s);
}

}  // namespace

long long planBeamSelect(BeamParams& p, LogitType type, void* base)
{
    (void)type;
    p.segs = 1;
    const long long items = (long long)p.groups * p.beams * p.segs;
    char* c = static_cast<char*>(base);
    p.sum = reinterpret_cast<double*>(c);
    p.keys = reinterpret_cast<unsigned long long*>(c + items * 8);
    p.top = reinterpret_cast<float*>(c + items * 8 * (1 + p.width));
    return items * (8 * (1 + p.width) + 4);
}

void launchBeamSelect(const BeamParams& p, LogitType type, cudaStream_t s)
{
    if (type == LOGITS_F32)
        launchSelectWidth<float>(p, s);
    else if (type == LOGITS_BF16)
        launchSelectWidth<__nv_bfloat16>(p, s);
    else
        launchSelectWidth<__half>(p, s);
}

void launchJointSelect(const BeamParams& p, LogitType type, cudaStream_t s)
{
    if (type == LOGITS_F32)
        jointSelectKernel<float><<<p.groups, MERGE_THREADS, 0, s>>>(p);
    else if (type == LOGITS_BF16)
        jointSelectKernel<__nv_bfloat16><<<p.groups, MERGE_THREADS, 0, s>>>(p);
    else
        jointSelectKernel<__half><<<p.groups, MERGE_THREADS, 0, s>>>(p);
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
