// paged_split.cuh -- how the paged attention kernels cut their work: tiles of
// 2^tile_shift rows of one (sequence, kv head, group of q heads), all tiles of
// a call in one list, an equal share of it to every CTA.  What a segment's
// start costs a CTA (q, the first maxima, the result) counts as seg_cost
// tiles, so that CTAs with many short segments get fewer of them.
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

// the CTA's share of the list, portion by portion.  A segment is seg_cost
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

// A CTA's share: units before each chunk of sequences, their total T, the
// first of CTA i's units (floor(i T / G)) as (sequence, head, unit).
template <int THREADS>
struct Share {
    long long scan[THREADS], off;
    int b0;
};
template <int THREADS>
__device__ __forceinline__ void share_of(const PagedAttendArgs &a, int segs, Share<THREADS> &sh, Walk &w, long long &T,
                                         long long &G) {
    constexpr int PER = THREADS / 32;
    const int tid = threadIdx.x, lane = tid & 31, n = a.kv.n_seqs;
    const int per = (n + THREADS - 1) / THREADS, lo = min(n, tid * per), hi = min(n, lo + per);
    long long mine = 0;
    for (int b = lo; b < hi; b++) mine += static_cast<long long>(Seq(a, b, blockIdx.x == 0).nt + a.seg_cost) * segs;
    sh.scan[tid] = mine;
    __syncthreads();
    if (tid < 32) {   // inclusive scan of the chunks, PER of them per lane
        long long v[PER], run = 0;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            run += sh.scan[lane * PER + i];
            v[i] = run;
        }
        long long x = run;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long u = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += u;
        }
#pragma unroll
        for (int i = 0; i < PER; i++) sh.scan[lane * PER + i] = v[i] + x - run;
    }
    __syncthreads();
    T = sh.scan[THREADS - 1];
    G = min(static_cast<long long>(gridDim.x), T);
    const long long i = blockIdx.x, at = i < G ? mul_div(i, T, G) : 0, end = i < G ? mul_div(i + 1, T, G) : 0;
    const long long before = sh.scan[tid] - mine;
    if (mine > 0 && at >= before && at < before + mine) {
        long long off = at - before;
        int b = lo;
        for (; b < hi; b++) {
            const long long nb = static_cast<long long>(Seq(a, b, false).nt + a.seg_cost) * segs;
            if (off < nb) break;
            off -= nb;
        }
        sh.b0 = b;
        sh.off = off;
    }
    __syncthreads();
    w.b = sh.b0;
    w.nt = Seq(a, w.b, false).nt;
    w.seg = static_cast<int>(mul_div(1, sh.off, w.nt + a.seg_cost));
    w.u = static_cast<int>(sh.off - static_cast<long long>(w.seg) * (w.nt + a.seg_cost));
    w.at = at;
    w.end = end;
}

// For the finish, by the CTA that has a cut segment's last tile: the CTA of
// its first tile << 16 | portions; 0 for a segment that is one portion
__device__ __forceinline__ unsigned cut_of(const Walk &w, long long T, long long G) {
    if (w.t0 == 0) return 0;
    const long long n = (w.at - w.nt + 1) * G - 1;
    const int own0 = static_cast<int>(T * G < (1ll << 31) ? static_cast<unsigned>(n) / static_cast<unsigned>(T) : n / T);
    return static_cast<unsigned>(own0) << 16 | (blockIdx.x - own0 + 1);
}
// where a portion's (max, sum, O) go: CTA i's portion that begins its segment
// to slot 2 i + 1, any other to slot 2 i.  O is [heads][pitch], then maxima
// and sums from kAttendPart - 32 on.
__device__ __forceinline__ float *part_at(const PagedAttendArgs &a, int cta, bool first) {
    return a.part + (2ll * cta + (first ? 1 : 0)) * kAttendPart;
}

}  // namespace
}  // namespace styx
