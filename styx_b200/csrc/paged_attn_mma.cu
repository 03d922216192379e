// paged_attn_mma.cu -- attention of one new token per sequence over a paged
// f16 / bf16 KV cache on the tensor cores (styx_paged_attend, head_dim up to
// 128, pages of 16 rows or more).
//
// Per kv head the step is two products whose long side is the rows:
//   S^T = K Q^T     [rows x heads],     O^T = V^T P^T     [head_dim x heads]
// with 16 rows (16 elements of head_dim) as M of mma.m16n8k16 and eight q
// heads as N: K and V are the A operands as they lie in memory, nothing is
// padded to a query tile, and eight heads of a kv head cost half of what
// they would as rows.  A row is 512 bytes (16 bits, head_dim 128) and, with
// eight heads, 2 (f16) or 3 (bf16) MMAs: a fifth of the rate of mma.sync when
// the rows come at HBM's.
//
// Precision.  q and p are f32 while K and V have 8 (bf16) or 11 (f16)
// significant bits, so q and p are split into 3 or 2 terms of the cache's
// type that add up to 24 / 22 bits; products are exact, sums f32.  The MMA
// cuts its sums off instead of rounding them, an error to one side that grows
// with every tile added to one accumulator (3.7e-6 of the output over 1800
// rows), so O is added up by the FMA units: tile by tile in registers, or
// (teams with shares of their own, whose q's place in shared memory is free
// by then; 16 heads 122 us otherwise) kSum tiles at a time in shared memory.
//
// A warp takes 16 rows at a time for itself; with more than eight q heads per
// kv head, two warps share them, eight heads each.  Copies (cp.async, 4 KB of
// K or V, contiguous in the page) go round a ring of the team's own, so that
// nobody else waits and 160 KB per SM are in flight.  The maximum that a row
// is measured against moves only when a score passes it by 2^8.  Each team
// has a share of the tile list and writes a cut segment's part from its
// registers; with few segments the CTA's teams take one share's tiles in turn
// and join in shared memory, so that a segment has an eighth of the parts.
// The next portion's first copies, its q ahead of them and its pages looked
// up together, are issued before the last one's result is written.
//
// Measured (B200): one sequence of 131071 f16 rows, 32 / 4 heads of 128, 268 MB
// in 50 us (5.3 TB/s; DRAM 66 % busy, tensor pipe 19 %, issue 34 %); twice as
// many rows 5.7 to 5.9 TB/s, what cp.async reaches here.  Bound by HBM with up
// to eight heads per kv head.  With 16 (bf16, 64 ragged sequences, 549 MB) 117
// us, bound by the latency of eight warps' MMAs and exchanges: as CTAs with
// one share 133 (125 with sums inside the MMA, then twelve warps 130, sixteen, whose registers spill, 151);
// one warp with all 16 heads 175; a branch around each MMA step (head_dim as a
// variable) 145; chains of MMAs half as long change nothing.  32 ragged bf16
// sequences of up to 4096 rows, 139 MB, 33.5 us: launch, share and first rows
// cost 4 us, a portion's end 2 us, the finish 3.
#include <cuda_runtime.h>

#include <cstdint>

#include "paged_split.cuh"

namespace styx {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kRows = 16;                      // rows of a tile
constexpr int kUnit = kRows * 256;             // K or V of them, 256-byte rows (head_dim 128)
constexpr int kUnits = 48;                     // of all rings
constexpr int kRing = kUnits * kUnit;
constexpr int kPad = 132;                      // floats of a head's q in shared memory: no two heads on one bank
constexpr int kQ = 8 * kPad * 4;               // q of eight heads
constexpr int kJoin = kWarps * 4 * kPad * 4;   // JOINT: four heads' results of every warp
constexpr int kRest = kWarps * kQ;             // beside the rings: q of every warp; JOINT: q, two buffers, and the join's
static_assert(kRest >= 2 * 2 * kQ + kJoin && kQ >= 32 * 32 * 4, "JOINT fits; O of a warp fits its q's place");
constexpr int kSum = 16;                       // tiles that the MMAs add up by themselves (a power of two)
constexpr float kSlack = 8.f;                  // log2 units a score may pass the maximum by

__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool on) {   // off: zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void ldm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldm4t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {   // of the 8 x 8 matrix that the warp holds
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
template <bool BF>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (BF)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// the same onto zeros
template <bool BF>
__device__ __forceinline__ void mma0(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (BF)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

// a pair of values (low half: x) as sums of terms of the cache's type, largest
// first.  bf16: the f32's 24 significant bits cut into 8 + 8 + 8, exactly;
// f16: rounded to 11, the rest rounded to 11.
template <bool BF>
__device__ __forceinline__ void split2(float x, float y, uint32_t (&t)[BF ? 3 : 2]) {
    if constexpr (BF) {
        uint32_t a = __float_as_uint(x), b = __float_as_uint(y);
#pragma unroll
        for (int i = 0; i < 3; i++) {
            t[i] = __byte_perm(a, b, 0x7632);
            const uint32_t c = __float_as_uint(__uint_as_float(a) - __uint_as_float(a & 0xFFFF0000u));
            const uint32_t d = __float_as_uint(__uint_as_float(b) - __uint_as_float(b & 0xFFFF0000u));
            a = c;
            b = d;
        }
    } else {
        const __half2 h = __floats2half2_rn(x, y);
        const float2 f = __half22float2(h);
        const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
        t[0] = *reinterpret_cast<const uint32_t *>(&h);
        t[1] = *reinterpret_cast<const uint32_t *>(&l);
    }
}

// a portion of the worker's share: its rows [lo, hi) of one segment, from base
// (lo rounded down to 16) on STEP rows at a time
template <int STEP>
struct Part {
    int b, j, g0, ng, lo, hi, base, iters;
    long long h0;
    const int32_t *table;
    __device__ __forceinline__ void set(const PagedAttendArgs &a, const Walk &wk, int groups, int nh) {
        const Seq s(a, wk.b, false);
        b = wk.b;
        j = wk.seg / groups;
        g0 = (wk.seg - j * groups) * nh;
        ng = min(nh, a.gqa - g0);
        h0 = static_cast<long long>(b) * a.n_heads + j * a.gqa + g0;
        table = a.kv.table + static_cast<long long>(b) * a.kv.table_stride;
        lo = max(s.first, (s.tile0 + wk.t0) << a.tile_shift);
        hi = static_cast<int>(min(static_cast<long long>(s.n), static_cast<long long>(s.tile0 + wk.t1) << a.tile_shift));
        base = lo & ~(kRows - 1);
        iters = hi > lo ? (hi - base + STEP - 1) / STEP : 0;
    }
};

// JOINT: the CTA's teams take the tiles of one share in turn and join their
// results at a portion's end; else each team has a share of its own.
// TEAM: warps that share a tile, eight q heads each; KS: 16-element steps of a
// row (what head_dim leaves of them is zeros)
template <bool BF, int TEAM, int KS, bool JOINT>
__global__ void __launch_bounds__(kThreads, 1) k_attend_mma(PagedAttendArgs a) {
    constexpr int TERMS = BF ? 3 : 2, NH = 8 * TEAM, TEAMS = kWarps / TEAM, S = kUnits / TEAMS, STEP = JOINT ? kRows * TEAMS : kRows;
    __shared__ float s_m[JOINT ? kWarps : 1][8], s_l[JOINT ? kWarps : 1][8], s_L[NH];
    extern __shared__ __align__(256) uint8_t smem[];   // (rows are swizzled by xor of address bits 4 to 7)
    const PagedKv &kv = a.kv;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, hd = kv.hd;
    const int team = warp / TEAM, in = warp % TEAM;   // in: which eight heads
    const int lr = lane >> 2, lc = lane & 3;   // of the fragments: row (B: column), pair of columns
    const int groups = (a.gqa + NH - 1) / NH, segs = kv.n_kv * groups;
    long long T, G;
    Walk wk;
    pdl_trigger();
    pdl_wait();
    // (neighbouring shares on different SMs: few tiles spread over all of them)
    const int worker = JOINT ? blockIdx.x : team * gridDim.x + blockIdx.x;
    share_of(a, segs, worker, wk, T, G);
    const uint32_t ring = smem_addr(smem) + team * S * kUnit;
    uint8_t *const rest = smem + kRing;
    float *sq = reinterpret_cast<float *>(rest + (JOINT ? 0 : warp * kQ));   // the portion's q, the CTA's or the warp's heads
    float *so = reinterpret_cast<float *>(rest + 4 * kQ);                    // JOINT: the join's buffer
    const float l2 = a.scale * 1.4426950408889634f;   // scores in units of log2
    auto team_sync = [&] {
        if constexpr (TEAM == 1) __syncwarp();
        else asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "n"(32 * TEAM) : "memory");
    };

    Part<STEP> P{};
    const int mine = JOINT ? team * kRows : 0;   // the team's rows of a step
    // ---------------- the ring: units K(0), V(0), K(1), ... of the team's tiles
    const bool col = (lane & 15) < hd / 8;
    // the lane's copies of a unit: rows at_row + 2 TEAM i, swizzled chunk lane % 16
    const int at_row = 2 * in + (lane >> 4), at_src = (at_row * hd + (col ? lane & 15 : 0) * 8) * 2;
    const uint32_t at_dst = ring + at_row * 256 + (((lane & 15) ^ at_row) << 4);
    int slot = 0;                     // of the next unit to be used
    unsigned seen = 0;                // bit s: slot s holds a tile of which rows are seen
    int kpage = -1, vpage = -1;       // the page of the next K, V to be copied; -1: none
    auto page_of = [&](int it) {
        const int r = P.base + it * STEP + mine;
        return it < P.iters && r < P.hi ? ld_now(P.table + (r >> kv.page_shift)) : -1;
    };
    // copies of K or V of tile `it` in a page into slot s; rows outside [lo, hi) are zeros, a page outside the pool is reported
    auto issue = [&](bool is_v, int it, int s, int page) {
        const int r0 = P.base + it * STEP + mine;
        const bool some = it < P.iters && r0 < P.hi, ok = some && static_cast<unsigned>(page) < static_cast<unsigned>(kv.n_pages);
        if (some && !ok && lane == 0) atomicExch(kv.err, kErrBadPos);
        if (ok) {
            const long long at = page * kv.page_stride + static_cast<long long>((P.j << kv.page_shift) +
                                                                                (r0 & ((1 << kv.page_shift) - 1))) * hd;
            const uint8_t *src = static_cast<const uint8_t *>(is_v ? kv.v : kv.k) + at * 2 + at_src;
            const unsigned first = r0 + at_row - P.lo, rows = P.hi - P.lo;
#pragma unroll
            for (int r = 0; r < kRows; r += 2 * TEAM)
                copy16((at_dst ^ ((r & 7) << 4)) + s * kUnit + r * 256, src + 2 * r * hd, col && first + r < rows);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        seen = ok ? seen | (1u << s) : seen & ~(1u << s);
    };
    auto start = [&] {                // a portion's first copies: q, then S - 1 units
        P.set(a, wk, groups, NH);
        int pages[S / 2];
#pragma unroll
        for (int i = 0; i < S / 2; i++) pages[i] = page_of(i);
        kpage = page_of(S / 2);
        vpage = pages[S / 2 - 1];
        const int per = hd / 4;
        if constexpr (JOINT) {
            sq = reinterpret_cast<float *>(rest + (reinterpret_cast<uint8_t *>(sq) == rest ? 2 * kQ : 0));
            for (int i = tid; i < P.ng * per; i += kThreads) {
                const int h = i / per, c = i - h * per;
                copy16(smem_addr(sq + h * kPad + 4 * c), a.q + (P.h0 + h) * hd + 4 * c, true);
            }
        } else {
            for (int i = lane; i < min(8, P.ng - 8 * in) * per; i += 32) {
                const int h = i / per, c = i - h * per;
                copy16(smem_addr(sq + h * kPad + 4 * c), a.q + (P.h0 + 8 * in + h) * hd + 4 * c, true);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        int s = slot;
#pragma unroll
        for (int u = 0; u < S - 1; u++) {
            issue(u & 1, u / 2, s, pages[u / 2]);
            s = s + 1 == S ? 0 : s + 1;
        }
    };
    // unit (it, is_v) is there for the whole team, and the copies of the one S - 1 later are on their way, into the
    // slot that the team has just read; returns the slot
    auto advance = [&](bool is_v, int it) {
        asm volatile("cp.async.wait_group %0;" ::"n"(S - 2) : "memory");
        team_sync();
        const int now = slot;
        slot = slot + 1 == S ? 0 : slot + 1;
        static_assert(S % 2 == 0, "V follows K");
        const int s = now == 0 ? S - 1 : now - 1;
        if (is_v) {
            issue(false, it + S / 2, s, kpage);
            vpage = kpage;
            kpage = page_of(it + S / 2 + 1);
        } else {
            issue(true, it + S / 2 - 1, s, vpage);
        }
        return now;
    };

    bool have = wk.next(a, segs);
    if (have) start();
    while (have) {
        asm volatile("cp.async.wait_group %0;" ::"n"(S - 1) : "memory");
        // q is there; the last join's buffers are free again
        if constexpr (JOINT) __syncthreads();
        else __syncwarp();
        // ---------------- q as B fragments, in terms.  f16 has few exponents: a head's largest |q| is brought to
        // [2^9, 2^10), and fh says what its column of S is in units of its terms
        uint32_t qf[KS][TERMS][2];
        float fh[2];
        {
            const int h = 8 * in + lr;
            const float *q = sq + (JOINT ? h : lr) * kPad + 2 * lc;
            float2 v[KS][2];
            float mx = 0.f;
#pragma unroll
            for (int k = 0; k < KS; k++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int d = 16 * k + 8 * i;
                    v[k][i] = make_float2(0.f, 0.f);
                    if (h < P.ng && d < hd) {
                        const float2 x = *reinterpret_cast<const float2 *>(q + d);
                        v[k][i] = make_float2(x.x * l2, x.y * l2);
                    }
                    mx = fmaxf(mx, fmaxf(fabsf(v[k][i].x), fabsf(v[k][i].y)));
                }
            float up = 1.f, down = 1.f;
            if constexpr (!BF) {
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                const int e = max(-110, min(110, static_cast<int>(__float_as_uint(mx) >> 23) - 127 - 9));
                up = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
                down = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
            }
            fh[0] = __shfl_sync(0xffffffffu, down, 8 * lc);        // heads 2 lc, 2 lc + 1 of the eight
            fh[1] = __shfl_sync(0xffffffffu, down, 8 * lc + 4);
#pragma unroll
            for (int k = 0; k < KS; k++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    uint32_t t[TERMS];
                    split2<BF>(v[k][i].x * up, v[k][i].y * up, t);
#pragma unroll
                    for (int z = 0; z < TERMS; z++) qf[k][z][i] = t[z];
                }
        }
        float m[2] = {kNone, kNone}, l[2] = {0.f, 0.f}, o[KS][4];
#pragma unroll
        for (int t = 0; t < KS; t++) o[t][0] = o[t][1] = o[t][2] = o[t][3] = 0.f;
        float *const sum = sq + lane;          // !JOINT: the sums of whole kSum tiles, where q was
        if constexpr (!JOINT) __syncwarp();
        const int hh = 8 * in + 2 * lc;        // the lane's heads of the group: hh, hh + 1
        float *scores = a.scores + (static_cast<long long>(P.b) * kv.n_kv + P.j) *
                                       (static_cast<long long>(kv.max_pages) << kv.page_shift) * a.gqa + P.g0 + hh;
        for (int it = 0; it < P.iters; it++) {
            const int r0 = P.base + it * STEP + mine + lr;   // the lane's rows: r0, r0 + 8
            const int kslot = advance(false, it);
            const bool live = (seen >> kslot) & 1;
            const bool in0 = r0 >= P.lo && r0 < P.hi, in1 = r0 + 8 >= P.lo && r0 + 8 < P.hi;
            uint32_t pf[TERMS][2];
            if (live) {
                // ---------------- S^T: row lr (+ 8), heads 2 lc, + 1
                float s[TERMS][4];
#pragma unroll
                for (int z = 0; z < TERMS; z++) s[z][0] = s[z][1] = s[z][2] = s[z][3] = 0.f;
                const uint32_t kt = ring + kslot * kUnit + (lane & 15) * 256 + (((lane >> 4) ^ (lane & 7)) << 4);
#pragma unroll
                for (int k = 0; k < KS; k++) {
                    uint32_t A[4];
                    ldm4(kt ^ (k << 5), A);
#pragma unroll
                    for (int z = 0; z < TERMS; z++) mma<BF>(s[z], A, qf[k][z][0], qf[k][z][1]);
                }
                const bool on[2] = {in0, in1};
                float x[4];                    // (row lr: heads 0, 1; row lr + 8: heads 0, 1)
                bool up = false;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    float y = s[0][i] + s[1][i];
                    if constexpr (TERMS == 3) y = s[0][i] + (s[1][i] + s[TERMS - 1][i]);
                    x[i] = on[i >> 1] ? (BF ? y : y * fh[i & 1]) : -INFINITY;
                    up |= x[i] > m[i & 1] + kSlack;
                }
                if (a.acc_out)
#pragma unroll
                    for (int i = 0; i < 2; i++)
                        if (on[i]) {
                            float *sc = scores + static_cast<long long>(r0 + 8 * i) * a.gqa;
                            if (hh < P.ng) sc[0] = x[2 * i];
                            if (hh + 1 < P.ng) sc[1] = x[2 * i + 1];
                        }
                if (__any_sync(0xffffffffu, up)) {
                    // new maxima over the sixteen rows; what was summed against the old ones is rescaled
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        float v = fmaxf(x[e], x[2 + e]);
                        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
                        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
                        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
                        v = fmaxf(v, m[e]);
                        const float f = ex2(m[e] - v);
                        m[e] = v;
                        l[e] *= f;
#pragma unroll
                        for (int t = 0; t < KS; t++) {
                            o[t][e] *= f;
                            o[t][2 + e] *= f;
                            if (!JOINT && it >= kSum) {
                                sum[(4 * t + e) * 32] *= f;
                                sum[(4 * t + 2 + e) * 32] *= f;
                            }
                        }
                    }
                }
                // ---------------- P^T as B fragments: eight rows by eight heads, transposed across the warp
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const float p0 = on[i] ? ex2(x[2 * i] - m[0]) : 0.f, p1 = on[i] ? ex2(x[2 * i + 1] - m[1]) : 0.f;
                    l[0] += p0;
                    l[1] += p1;
                    uint32_t t[TERMS];
                    // f16: p up to 2^8 is carried as p * 2^7, so that the second term of a small p keeps its bits
                    split2<BF>(BF ? p0 : p0 * 128.f, BF ? p1 : p1 * 128.f, t);
#pragma unroll
                    for (int z = 0; z < TERMS; z++) pf[z][i] = transposed(t[z]);
                }
            } else if (a.acc_out) {            // rows of a page outside the pool
                if (in0 && hh < P.ng) scores[static_cast<long long>(r0) * a.gqa] = -INFINITY;
                if (in0 && hh + 1 < P.ng) scores[static_cast<long long>(r0) * a.gqa + 1] = -INFINITY;
                if (in1 && hh < P.ng) scores[static_cast<long long>(r0 + 8) * a.gqa] = -INFINITY;
                if (in1 && hh + 1 < P.ng) scores[static_cast<long long>(r0 + 8) * a.gqa + 1] = -INFINITY;
            }
            const int vslot = advance(true, it);
            if (live) {
                // ---------------- O^T += V^T P^T
                const uint32_t vt = ring + vslot * kUnit + ((lane & 7) + ((lane >> 4) << 3)) * 256 +
                                    ((((lane >> 3) & 1) ^ (lane & 7)) << 4);
#pragma unroll
                for (int t = 0; t < KS; t++) {
                    uint32_t A[4];
                    ldm4t(vt ^ (t << 5), A);
                    if constexpr (JOINT) {
                        float d[4];
                        mma0<BF>(d, A, pf[TERMS - 1][0], pf[TERMS - 1][1]);
#pragma unroll
                        for (int z = TERMS - 2; z >= 0; z--) mma<BF>(d, A, pf[z][0], pf[z][1]);
#pragma unroll
                        for (int i = 0; i < 4; i++) o[t][i] += d[i];
                    } else {
#pragma unroll
                        for (int z = TERMS - 1; z >= 0; z--) mma<BF>(o[t], A, pf[z][0], pf[z][1]);
                    }
                }
            }
            if (!JOINT && (it & (kSum - 1)) == kSum - 1) {
#pragma unroll
                for (int t = 0; t < KS; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        sum[(4 * t + i) * 32] = it < kSum ? o[t][i] : sum[(4 * t + i) * 32] + o[t][i];
                        o[t][i] = 0.f;
                    }
            }
        }
        if (!JOINT && P.iters >= kSum)
#pragma unroll
            for (int t = 0; t < KS; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) o[t][i] += sum[(4 * t + i) * 32];
        // ---------------- the portion's end: the next one's first copies, then the result
        const int ng = P.ng;
        const long long h0 = P.h0;
        const bool first = wk.t0 == 0, whole = first && wk.t1 == wk.nt;
        if (wk.t1 == wk.nt && (JOINT ? tid == 0 : in == 0 && lane == 0)) a.cnt[static_cast<long long>(wk.b) * segs + wk.seg] = cut_of(wk, worker, T, G);
        have = wk.next(a, segs);
        team_sync();
        if (have) start();
        float *part = part_at(a, worker, first);
#pragma unroll
        for (int e = 0; e < 2; e++) {
            l[e] += __shfl_xor_sync(0xffffffffu, l[e], 4);
            l[e] += __shfl_xor_sync(0xffffffffu, l[e], 8);
            l[e] += __shfl_xor_sync(0xffffffffu, l[e], 16);
        }
        auto put_sums = [&](int h, float M, float L) {
            if (!whole) {
                part[a.part_floats - 32 + h] = M;
                part[a.part_floats - 16 + h] = L;
                return;
            }
            if (a.lse) a.lse[h0 + h] = lse_of(M, L);
            if (a.acc_out) {
                a.ml[2 * (h0 + h)] = M;
                a.ml[2 * (h0 + h) + 1] = L;
            }
        };
        constexpr float kUp = BF ? 1.f : 0x1p-7f;   // (f16: p was carried times 2^7)
        if constexpr (!JOINT) {
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int h = hh + e;
                if (h >= ng) continue;
                const float r = (whole ? inverse_sum(l[e]) : 1.f) * kUp;
                float *to = whole ? a.out + (h0 + h) * hd : part + h * 128;
#pragma unroll
                for (int t = 0; t < KS; t++)
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const int c = 16 * t + 8 * i + lr;
                        if (c < hd) to[c] = o[t][2 * i + e] * r;
                    }
                if (lr == 0) put_sums(h, m[e], l[e]);
            }
        } else {
            if (lr == 0)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    s_m[warp][2 * lc + e] = m[e];
                    s_l[warp][2 * lc + e] = l[e];
                }
#pragma unroll
            for (int n = 0; n < 2; n++) {          // four heads of every warp at a time
                if (lc >> 1 == n)
#pragma unroll
                    for (int t = 0; t < KS; t++)
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            so[(warp * 4 + 2 * (lc & 1) + (i & 1)) * kPad + 16 * t + lr + 8 * (i >> 1)] = o[t][i] * kUp;
                __syncthreads();
                if (n == 0) {
                    if (tid < NH) {
                        float M = kNone, L = 0.f;
                        for (int w = 0; w < TEAMS; w++) M = fmaxf(M, s_m[w * TEAM + tid / 8][tid & 7]);
                        for (int w = 0; w < TEAMS; w++) {
                            float &mw = s_m[w * TEAM + tid / 8][tid & 7];
                            mw = ex2(mw - M);
                            L += s_l[w * TEAM + tid / 8][tid & 7] * mw;
                        }
                        s_L[tid] = L;
                        if (tid < ng) put_sums(tid, M, L);
                    }
                    __syncthreads();
                }
                for (int i = tid; i < 4 * TEAM * hd; i += kThreads) {
                    const int g = i / hd, c = i - g * hd, e = g / 4, h4 = g & 3, h = 8 * e + 4 * n + h4;
                    if (h >= ng) continue;
                    float v = 0.f;
#pragma unroll
                    for (int w = 0; w < TEAMS; w++) v += so[((w * TEAM + e) * 4 + h4) * kPad + c] * s_m[w * TEAM + e][4 * n + h4];
                    if (whole) a.out[(h0 + h) * hd + c] = s_L[h] == 0.f ? 0.f : v / s_L[h];
                    else part[h * 128 + c] = v;
                }
                if (n == 0) __syncthreads();
            }
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

template <bool BF, int TEAM, int KS, bool JOINT>
cudaError_t launch(PagedAttendArgs a, int sms, cudaStream_t st) {
    constexpr int smem = kRing + kRest;
    const cudaError_t e = allow_smem<k_attend_mma<BF, TEAM, KS, JOINT>>(smem);
    if (e != cudaSuccess) return e;
    // (a segment of up to 128 rows whole: it needs no join, the call no second kernel)
    a.tile_shift = JOINT || static_cast<long long>(a.kv.max_pages) << a.kv.page_shift <= 128 ? 7 : 4;
    a.seg_cost = JOINT ? 3 : 4;
    a.part_floats = attend_part(8 * TEAM, 128);
    const int ctas = attend_grid(a, 8 * TEAM, sms);
    a.workers = JOINT ? ctas : ctas * (kWarps / TEAM);
    const cudaError_t e2 = launch_pdl(k_attend_mma<BF, TEAM, KS, JOINT>, dim3(ctas), dim3(kThreads), smem, st, a);
    return e2 != cudaSuccess ? e2 : launch_attend_finish(a, 8 * TEAM, 128, st);
}
template <bool BF, int TEAM>
cudaError_t launch_t(const PagedAttendArgs &a, int sms, cudaStream_t st) {
    // Segments no more than SMs: a CTA's warps together on one of them (one sequence of 131071 rows 50 us, each warp
    // for itself 68, whose 296 results per segment take long to join; 32 ragged ones 33.5 against 35).  More: each team
    // for itself, so that a segment's start and end stop nobody else (64 sequences of up to 512 rows 15 us against 19,
    // 128 of up to 1024 with 8 kv heads 57 against 63, 64 of up to 8192 with 64 / 4 heads 117 against 133; of up to
    // 2048 with 32 / 4 heads 37 against 35).
    const long long segs = static_cast<long long>(a.kv.n_seqs) * a.kv.n_kv * ((a.gqa + 8 * TEAM - 1) / (8 * TEAM));
    if (a.kv.hd <= 64) return segs <= sms ? launch<BF, TEAM, 4, true>(a, sms, st) : launch<BF, TEAM, 4, false>(a, sms, st);
    return segs <= sms ? launch<BF, TEAM, 8, true>(a, sms, st) : launch<BF, TEAM, 8, false>(a, sms, st);
}

}  // namespace

uint64_t attend_mma_parts(int gqa, int sms) {
    const int team = gqa <= 8 ? 1 : 2;
    return 2ull * sms * (kWarps / team) * attend_part(8 * team, 128) * 4;
}

cudaError_t launch_attend_mma(const PagedAttendArgs &a, int sms, cudaStream_t st) {
    if (a.kv.dtype == STYX_BF16) return a.gqa <= 8 ? launch_t<true, 1>(a, sms, st) : launch_t<true, 2>(a, sms, st);
    return a.gqa <= 8 ? launch_t<false, 1>(a, sms, st) : launch_t<false, 2>(a, sms, st);
}

}  // namespace styx
