// paged_split.cuh -- how the paged attention kernels cut their work: tiles of
// 2^tile_shift rows of one (sequence, kv head, group of q heads), all tiles of
// a call in one list, an equal share of it to every worker (a CTA, or a team of
// warps).  What a segment's start costs it (q, the first maxima, the result)
// counts as seg_cost tiles, so that those with many short segments get fewer.
#pragma once

#include "paged.cuh"

namespace styx {
namespace {

constexpr float kNone = -3e38f;            // maximum of no scores: finite, so that differences stay numbers

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A softmax's sum is 0 where no row was seen, and only there: a row's weight
// against the maximum is 1 for one of them.  NaN (of a NaN in q or K, or of a
// score of +inf) is neither, and goes to the output.
__device__ __forceinline__ float inverse_sum(float sum) { return sum == 0.f ? 0.f : 1.f / sum; }
__device__ __forceinline__ float lse_of(float max, float sum) {   // max in units of log2
    return sum == 0.f ? -INFINITY : max * 0.6931471805599453f + logf(sum);
}

// rows of a sequence that are seen, and its tiles (an empty one counts one
// tile, so that somebody writes its zeros)
struct Seq {
    int n, first, tile0, nt;
    __device__ __forceinline__ Seq(const PagedAttendArgs &a, int b, bool report) {
        n = paged_len(a.kv, b, report);
        first = a.window > 0 && a.window < n ? n - a.window : 0;
        tile0 = first >> a.tile_shift;
        nt = max(1, static_cast<int>((n + (1ll << a.tile_shift) - 1) >> a.tile_shift) - tile0);
    }
};

// a worker's share of the list, portion by portion.  A segment is seg_cost
// empty units, then its tiles.
struct Walk {
    int b, seg, u, nt;             // sequence, (kv head, group) in it, next unit of seg_cost + nt
    long long at, end;             // global unit numbers
    int t0, t1;                    // the portion: tiles [t0, t1) of the segment
    __device__ __forceinline__ bool next(const PagedAttendArgs &a, int segs) {
        while (at < end) {
            if (u == a.seg_cost + nt) {
                u = 0;
                if (++seg == segs) {
                    seg = 0;
                    if (++b >= a.kv.n_seqs) {   // (lengths that changed during the call)
                        end = at;
                        return false;
                    }
                    nt = Seq(a, b, false).nt;
                }
            }
            const int u1 = static_cast<int>(min(static_cast<long long>(a.seg_cost + nt), u + (end - at)));
            t0 = max(0, u - a.seg_cost);
            t1 = max(0, u1 - a.seg_cost);
            at += u1 - u;
            u = u1;
            if (t1 > t0) return true;
        }
        return false;
    }
};


// x y / d, all below 2^31: a 32-bit division (a 64-bit one is some 300 clocks) where the product allows it
__device__ __forceinline__ long long mul_div(long long x, long long y, long long d) {
    const unsigned long long p = static_cast<unsigned long long>(x) * y;
    return p >> 32 ? static_cast<long long>(p / d) : static_cast<long long>(static_cast<unsigned>(p) / static_cast<unsigned>(d));
}

// A worker's share: the units of all sequences, T, and the first of worker i's
// (floor(i T / G)) as (sequence, head, unit).  Every warp finds it for itself,
// a run of sequences per lane: with the CTA's barriers it was twice as long.
__device__ __forceinline__ void share_of(const PagedAttendArgs &a, int segs, int worker, Walk &w, long long &T, long long &G) {
    const int lane = threadIdx.x & 31, n = a.kv.n_seqs;
    const int per = (n + 31) / 32, lo = min(n, lane * per), hi = min(n, lo + per);
    const bool report = blockIdx.x == 0 && threadIdx.x < 32;
    auto units = [&](int b, bool r) { return static_cast<long long>(Seq(a, b, r).nt + a.seg_cost) * segs; };
    long long mine = 0;
#pragma unroll 4
    for (int b = lo; b < hi; b++) mine += units(b, report);
    long long upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += u;
    }
    T = __shfl_sync(0xffffffffu, upto, 31);
    G = min(static_cast<long long>(a.workers), T);
    const long long i = worker, at = i < G ? mul_div(i, T, G) : 0, end = i < G ? mul_div(i + 1, T, G) : 0;
    const int src = __ffs(__ballot_sync(0xffffffffu, at < upto)) - 1;   // (at < T, so there is one)
    long long off = at - (upto - mine);
    int b = lo;
    if (lane == src)
        for (; b < hi - 1; b++) {
            const long long nb = units(b, false);
            if (off < nb) break;
            off -= nb;
        }
    w.b = __shfl_sync(0xffffffffu, b, src);
    off = __shfl_sync(0xffffffffu, off, src);
    w.nt = Seq(a, w.b, false).nt;
    w.seg = static_cast<int>(min(mul_div(1, off, w.nt + a.seg_cost), static_cast<long long>(segs - 1)));
    w.u = static_cast<int>(min(off - static_cast<long long>(w.seg) * (w.nt + a.seg_cost),
                               static_cast<long long>(w.nt + a.seg_cost)));   // (bounds: lengths that changed)
    w.at = at;
    w.end = end;
}

// For the finish, by the worker that has a cut segment's last tile: that of
// its first tile << 16 | portions; 0 for a segment that is one portion
__device__ __forceinline__ unsigned cut_of(const Walk &w, int worker, long long T, long long G) {
    if (w.t0 == 0) return 0;
    const long long n = (w.at - w.nt + 1) * G - 1;
    const int own0 = static_cast<int>(T * G < (1ll << 31) ? static_cast<unsigned>(n) / static_cast<unsigned>(T) : n / T);
    return static_cast<unsigned>(own0) << 16 | (worker - own0 + 1);
}
// where a portion's (max, sum, O) go: worker i's portion that begins its segment
// to slot 2 i + 1, any other to slot 2 i.  O is [heads][pitch], then maxima
// and sums from part_floats - 32 on.
__device__ __forceinline__ float *part_at(const PagedAttendArgs &a, int worker, bool first) {
    return a.part + (2ll * worker + (first ? 1 : 0)) * a.part_floats;
}

}  // namespace
}  // namespace styx
