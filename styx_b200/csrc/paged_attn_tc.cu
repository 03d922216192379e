// paged_attn_tc.cu -- attention of one new token per sequence over a paged
// f16 / bf16 KV cache on the tensor cores (styx_paged_attend, head_dim 64 to
// 128, pages of 16 rows or more).
//
// Per kv head the step is two products whose long side is the rows:
//   S^T = K Q^T     [rows x heads],     O^T = V^T P^T     [head_dim x heads]
// with 128 rows (head_dim) as M of tcgen05.mma and the kv head's q heads as
// N, so the cache's rows are the A operand straight from where TMA put them
// (K: K-major, V: M-major, both 128-byte swizzled) and nothing is
// transposed or padded to a query tile.
//
// Precision.  q and p are f32 while K and V have 8 (bf16) or 11 (f16)
// significant bits, so q and p are split into 3 or 2 terms of the cache's
// type that add up to 24 / 22 bits; the terms are further columns of N, the
// products are exact and the sums f32 in TMEM.  The wider N costs nothing:
// an instruction's time is its A operand's.
//
// The work is cut into tiles of 128 rows of one (sequence, kv head, group of
// NH q heads).  All tiles of the call form one list; CTA i of G takes the
// i-th G-th of it, so ragged lengths spread evenly over the SMs.  A portion
// (a CTA's consecutive tiles of one segment) ends in (max, sum, O) per head:
// written out where it is the whole segment, else to the workspace, and the
// CTA that finishes a segment's last portion joins them in order.  Which CTA
// that is does not change the result.
//
// Roles, linked by mbarriers with bounded waits: warps 0-3 softmax (thread =
// row of the tile; in the end thread = element of head_dim), warp 4 copies K,
// warp 5 copies V (a ring of 3 stages of 128 rows, 192 KB: more than the
// bytes in flight that HBM's latency needs), warp 6 issues the MMAs.  The
// maximum a row is measured against moves only when a score passes it by
// 2^8, so the accumulator is rescaled rarely and no tile waits for an exact
// running maximum; sums and exponentials are unaffected by which one is used.
#include <cuda_runtime.h>

#include <cstdint>

#include "paged.cuh"

namespace styx {
namespace {

constexpr int kTile = 128;                 // rows of a tile = M of both products
constexpr int kStages = 3;
constexpr int kHalfBytes = kTile * 128;    // 64 columns of a tile: 128-byte rows
constexpr int kSlotBytes = 2 * kHalfBytes; // K or V of a tile
constexpr int kThreads = 224;
constexpr int kWarpK = 4, kWarpV = 5, kWarpMma = 6;
constexpr uint32_t kTmemCols = 256, kColS = 64, kColO = 128;
constexpr float kSlack = 8.f;              // log2 units a score may pass the maximum by

template <bool BF, int NH>
struct Cfg {
    static constexpr int terms = BF ? 3 : 2;
    static constexpr int nb = (terms * NH + 15) / 16 * 16;   // N of the products (M 128: multiples of 16)
    static constexpr int q_bytes = 2 * nb * 128, p_bytes = 2 * nb * 128;
    static constexpr int smem = 2 * kStages * kSlotBytes + q_bytes + p_bytes + 1024;
    // term of a small p keeps its bits; bf16 has f32's range
};

// ------------------------------------------------------------ tensor-core helpers
// shared-memory operand, 128-byte swizzle, descriptor version 1.  K-major:
// sbo = bytes between groups of 8 rows.  M-major: lbo = bytes between blocks
// of 64 along M, sbo = bytes between groups of 8 along K.
__device__ __forceinline__ uint64_t desc_sw128(uint32_t addr, uint32_t lbo, uint32_t sbo) {
    uint64_t d = static_cast<uint64_t>((addr >> 4) & 0x3FFFu);
    d |= static_cast<uint64_t>((lbo >> 4) & 0x3FFFu) << 16;
    d |= static_cast<uint64_t>((sbo >> 4) & 0x3FFFu) << 32;
    d |= static_cast<uint64_t>(1) << 46;
    d |= static_cast<uint64_t>(2) << 61;
    return d;
}
// f32 accumulator, A and B both f16 or both bf16, M 128; a_mn: A is M-major
constexpr uint32_t idesc(bool bf, int n, bool a_mn) {
    return (1u << 4) | (bf ? (1u << 7) | (1u << 10) : 0u) | (a_mn ? 1u << 15 : 0u) |
           (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(kTile >> 4) << 24);
}
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t id, bool acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(id), "r"(static_cast<uint32_t>(acc)));
}
__device__ __forceinline__ void commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar))
                 : "memory");
}
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void ld8(uint32_t addr, float *v) {
    uint32_t r[8];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(addr));
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = __uint_as_float(r[j]);
}
__device__ __forceinline__ void st8(uint32_t addr, const float *v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr),
                 "r"(__float_as_uint(v[0])), "r"(__float_as_uint(v[1])), "r"(__float_as_uint(v[2])),
                 "r"(__float_as_uint(v[3])), "r"(__float_as_uint(v[4])), "r"(__float_as_uint(v[5])),
                 "r"(__float_as_uint(v[6])), "r"(__float_as_uint(v[7]))
                 : "memory");
}
// N columns of this thread's lane; the values are valid after the wait, which
// the compiler must not move their uses across
template <int N>
__device__ __forceinline__ void ld_cols(uint32_t addr, float (&v)[N]) {
    static_assert(N % 8 == 0, "columns by eights");
#pragma unroll
    for (int c = 0; c < N; c += 8) ld8(addr + c, v + c);
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int c = 0; c < N; c++) asm volatile("" : "+f"(v[c]));
}
__device__ __forceinline__ void tma3(void *dst, const CUtensorMap *map, int x, int y, int z, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
        "[%5];" ::"r"(smem_addr(dst)),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_addr(bar))
        : "memory");
}
__device__ __forceinline__ void wg_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
__device__ __forceinline__ bool wg_any(bool v) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\t"
        "barrier.cta.red.or.pred q, 1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r)
        : "r"(static_cast<uint32_t>(v))
        : "memory");
    return r != 0;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// v as a sum of terms of the cache's type, largest first
template <bool BF>
__device__ __forceinline__ void split(float v, uint16_t (&t)[BF ? 3 : 2]) {
    if constexpr (BF) {
        const __nv_bfloat16 a = __float2bfloat16_rn(v);
        const float r = v - __bfloat162float(a);
        const __nv_bfloat16 b = __float2bfloat16_rn(r);
        const __nv_bfloat16 c = __float2bfloat16_rn(r - __bfloat162float(b));
        t[0] = __bfloat16_as_ushort(a);
        t[1] = __bfloat16_as_ushort(b);
        t[2] = __bfloat16_as_ushort(c);
    } else {
        const __half a = __float2half_rn(v);
        t[0] = __half_as_ushort(a);
        t[1] = __half_as_ushort(__float2half_rn(v - __half2float(a)));
    }
}
// byte of (row n, element c of 128) of a K-major B operand [2][nb][64], swizzled
__device__ __forceinline__ uint32_t b_off(int nb, int n, int c) {
    return static_cast<uint32_t>((c >> 6) * nb * 128 + n * 128 + ((((c & 63) >> 3) ^ (n & 7)) << 4) + (c & 7) * 2);
}

struct Bars {
    uint64_t kfull[kStages], kempty[kStages], vfull[kStages], vempty[kStages];
    uint64_t sfull[2], pfull, odone, qfull, drain;
};

// rows of a sequence that are seen, and its tiles (an empty one counts one
// tile, so that somebody writes its zeros)
struct Seq {
    int n, first, tile0, nt;
    __device__ __forceinline__ Seq(const PagedAttendArgs &a, int b, bool report) {
        n = paged_len(a.kv, b, report);
        first = a.window > 0 && a.window < n ? n - a.window : 0;
        tile0 = first / kTile;
        nt = max(1, (n + kTile - 1) / kTile - tile0);
    }
};

// the CTA's share of the tile list, portion by portion
struct Walk {
    int b, seg, t, nt;             // sequence, (kv head, group) in it, next tile of nt
    long long at, end;             // global tile numbers
    int t0, t1;                    // the portion: tiles [t0, t1) of the segment
    __device__ __forceinline__ bool next(const PagedAttendArgs &a, int segs) {
        if (at >= end) return false;
        if (t == nt) {
            t = 0;
            if (++seg == segs) {
                seg = 0;
                b++;
                nt = Seq(a, b, false).nt;
            }
        }
        t0 = t;
        t1 = static_cast<int>(min(static_cast<long long>(nt), t + (end - at)));
        at += t1 - t0;
        t = t1;
        return true;
    }
};

template <bool BF, int NH>
__global__ void __launch_bounds__(kThreads, 1)
    k_attend_tc(PagedAttendArgs a, const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv) {
    using C = Cfg<BF, NH>;
    constexpr int NB = C::nb, TERMS = C::terms;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *sm = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
    uint8_t *sK = sm, *sV = sm + kStages * kSlotBytes, *sQ = sV + kStages * kSlotBytes, *sP = sQ + C::q_bytes;
    __shared__ Bars bars;
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort, s_b0, s_last;
    __shared__ long long s_off, s_scan[kThreads];
    __shared__ float s_red[4][16], s_f[16];
    const PagedKv &kv = a.kv;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int groups = (a.gqa + NH - 1) / NH, segs = kv.n_kv * groups;

    pdl_trigger();
    if (tid == 0) {
        for (int i = 0; i < kStages; i++) {
            mbar_init(&bars.kfull[i], 1);
            mbar_init(&bars.kempty[i], 1);
            mbar_init(&bars.vfull[i], 1);
            mbar_init(&bars.vempty[i], 1);
        }
        mbar_init(&bars.sfull[0], 1);
        mbar_init(&bars.sfull[1], 1);
        mbar_init(&bars.pfull, 128);
        mbar_init(&bars.odone, 1);
        mbar_init(&bars.qfull, 128);
        mbar_init(&bars.drain, 1);
        fence_mbar_init();
        s_abort = 0;
    }
    if (warp == kWarpMma) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&s_tmem)),
                     "r"(kTmemCols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    pdl_wait();

    // ---------------- the CTA's share: tiles before each chunk of sequences, total
    Walk w0;
    {
        const int per = (kv.n_seqs + kThreads - 1) / kThreads, lo = min(kv.n_seqs, tid * per), hi = min(kv.n_seqs, lo + per);
        long long mine = 0;
        for (int b = lo; b < hi; b++) mine += static_cast<long long>(Seq(a, b, blockIdx.x == 0).nt) * segs;
        s_scan[tid] = mine;
        __syncthreads();
        if (warp == 0) {   // inclusive scan of the kThreads chunks, seven per lane
            long long v[kThreads / 32], run = 0;
#pragma unroll
            for (int i = 0; i < kThreads / 32; i++) {
                run += s_scan[lane * (kThreads / 32) + i];
                v[i] = run;
            }
            long long x = run;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long u = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= o) x += u;
            }
#pragma unroll
            for (int i = 0; i < kThreads / 32; i++) s_scan[lane * (kThreads / 32) + i] = v[i] + x - run;
        }
        __syncthreads();
        const long long T = s_scan[kThreads - 1];
        const long long G = min(static_cast<long long>(gridDim.x), T);
        const long long at = blockIdx.x < G ? blockIdx.x * T / G : 0, end = blockIdx.x < G ? (blockIdx.x + 1) * T / G : 0;
        const long long before = s_scan[tid] - mine;
        if (mine > 0 && at >= before && at < before + mine) {
            long long off = at - before;
            int b = lo;
            for (; b < hi; b++) {
                const long long nb = static_cast<long long>(Seq(a, b, false).nt) * segs;
                if (off < nb) break;
                off -= nb;
            }
            s_b0 = b;
            s_off = off;
        }
        __syncthreads();
        w0.b = s_b0;
        w0.nt = Seq(a, w0.b, false).nt;
        w0.seg = static_cast<int>(s_off / w0.nt);
        w0.t = static_cast<int>(s_off - static_cast<long long>(w0.seg) * w0.nt);
        w0.at = at;
        w0.end = end;
    }
    const long long T = s_scan[kThreads - 1], G = min(static_cast<long long>(gridDim.x), T);
    const uint32_t tmem = s_tmem;
    Walk wk = w0;

    auto wait = [&](uint64_t *bar, uint32_t parity) {
        if (mbar_try_wait(bar, parity)) return true;
        const long long t0 = clock64();
        while (true) {
            if (mbar_try_wait_suspend(bar, parity)) return true;
            if (*reinterpret_cast<volatile int *>(&s_abort)) return false;
            if (clock64() - t0 > kSpinCycles) {
                atomicExch(kv.err, kErrWaitFull);
                *reinterpret_cast<volatile int *>(&s_abort) = 1;
                return false;
            }
        }
    };

    if (warp == kWarpK || warp == kWarpV) {
        // ---------------- copies: boxes of min(page, 128) rows x 64 columns
        const bool isv = warp == kWarpV;
        const CUtensorMap *map = isv ? &mv : &mk;
        uint8_t *ring = isv ? sV : sK;
        uint64_t *full = isv ? bars.vfull : bars.kfull, *empty = isv ? bars.vempty : bars.kempty;
        const int rb_shift = min(kv.page_shift, 7), rows = 1 << rb_shift, halves = kv.hd > 64 ? 2 : 1;
        const int boxes = (kTile >> rb_shift) * halves;   // <= 16
        const int pi = lane / halves, half = lane - pi * halves;
        int q = 0;
        bool live = true;
        while (live && wk.next(a, segs)) {
            const Seq s(a, wk.b, false);
            const int j = wk.seg / groups;
            const int32_t *table = kv.table + static_cast<long long>(wk.b) * kv.table_stride;
            for (int t = wk.t0; t < wk.t1; t++, q++) {
                const int st = q % kStages, use = q / kStages;
                const int r0 = (s.tile0 + t) * kTile + (pi << rb_shift);
                bool on = lane < boxes && r0 < s.n && r0 + rows > s.first;
                int page = 0;
                if (on) {
                    page = __ldg(table + (r0 >> kv.page_shift));
                    if (static_cast<unsigned>(page) >= static_cast<unsigned>(kv.n_pages)) {
                        if (!isv) atomicExch(kv.err, kErrBadPos);
                        on = false;
                    }
                }
                const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, on)) * static_cast<uint32_t>(rows) * 128u;
                if (use > 0 && !__all_sync(0xffffffffu, wait(&empty[st], static_cast<uint32_t>((use - 1) & 1)))) {
                    live = false;
                    break;
                }
                if (lane == 0) mbar_arrive_expect_tx(&full[st], bytes);
                __syncwarp();
                if (on)
                    tma3(ring + st * kSlotBytes + half * kHalfBytes + (pi << rb_shift) * 128, map, half * 64,
                         (j << kv.page_shift) + (r0 & ((1 << kv.page_shift) - 1)), page, &full[st]);
            }
        }
        // nothing of this warp's is still landing when the CTA ends
        for (int i = max(0, q - kStages); i < q; i++) mbar_wait(&full[i % kStages], static_cast<uint32_t>((i / kStages) & 1), nullptr, 0);
    } else if (warp == kWarpMma) {
        // ---------------- one thread issues the products
        if (lane == 0) {
            constexpr uint32_t id_s = idesc(BF, NB, false), id_o = idesc(BF, NB, true);
            const int ksteps = (kv.hd + 15) / 16;
            const uint32_t aK = smem_addr(sK), aV = smem_addr(sV), aQ = smem_addr(sQ), aP = smem_addr(sP);
            int q = 0, portion = 0;
            bool live = true;
            auto scores = [&](int i) {   // S of tile i (global number) into buffer i % 2
                const int st = i % kStages;
                if (!wait(&bars.kfull[st], static_cast<uint32_t>((i / kStages) & 1))) return false;
                fence_after();
                for (int k = 0; k < ksteps; k++) {
                    const uint32_t in = static_cast<uint32_t>(k & 3) * 32;
                    mma(tmem + (i & 1) * kColS,
                        desc_sw128(aK + st * kSlotBytes + (k >> 2) * kHalfBytes + in, 16, 1024),
                        desc_sw128(aQ + (k >> 2) * NB * 128 + in, 16, 1024), id_s, k > 0);
                }
                commit(&bars.kempty[st]);
                commit(&bars.sfull[i & 1]);
                return true;
            };
            while (live && wk.next(a, segs)) {
                const int nt = wk.t1 - wk.t0;
                if (!wait(&bars.qfull, static_cast<uint32_t>(portion & 1))) break;
                fence_after();
                live = scores(q);
                for (int t = 0; t < nt && live; t++, q++) {
                    if (t + 1 < nt && !(live = scores(q + 1))) break;
                    const int st = q % kStages;
                    if (!(live = wait(&bars.vfull[st], static_cast<uint32_t>((q / kStages) & 1)))) break;
                    if (!(live = wait(&bars.pfull, static_cast<uint32_t>(q & 1)))) break;
                    fence_after();
#pragma unroll
                    for (int k = 0; k < kTile / 16; k++)
                        mma(tmem + kColO, desc_sw128(aV + st * kSlotBytes + k * 2048, kHalfBytes, 1024),
                            desc_sw128(aP + (k >> 2) * NB * 128 + (k & 3) * 32, 16, 1024), id_o, t > 0 || k > 0);
                    commit(&bars.vempty[st]);
                    commit(&bars.odone);
                }
                portion++;
            }
            // every product issued here has completed before TMEM is freed
            commit(&bars.drain);
            mbar_wait(&bars.drain, 0u, nullptr, 0);
        }
        __syncwarp();
    } else {
        // ---------------- softmax: thread = row of the tile.  A wait that gave
        // up is not looked at here: every thread goes on to the end, so the
        // four warps stay together at their barriers (later waits return at
        // once, the results are void and the error word says so).
        const uint32_t lane_base = static_cast<uint32_t>(32 * warp) << 16;
        const float l2 = a.scale * 1.4426950408889634f;   // scores in units of log2
        const long long max_rows = static_cast<long long>(kv.max_pages) << kv.page_shift;
        int q = 0;
        while (wk.next(a, segs)) {
            const Seq s(a, wk.b, false);
            const int j = wk.seg / groups, g0 = (wk.seg - j * groups) * NH, ng = min(NH, a.gqa - g0);
            const long long h0 = static_cast<long long>(wk.b) * a.n_heads + j * a.gqa + g0;
            const int32_t *table = kv.table + static_cast<long long>(wk.b) * kv.table_stride;
            float fh[NH];          // what a column of S is in units of its terms
            {                      // Q: thread = element, split into terms
                float qv[NH];
#pragma unroll
                for (int h = 0; h < NH; h++) qv[h] = h < ng && tid < kv.hd ? __ldg(a.q + (h0 + h) * kv.hd + tid) * l2 : 0.f;
                if constexpr (!BF) {
                    // f16 has few exponents: every head's largest |q| is brought to [2^9, 2^10)
#pragma unroll
                    for (int h = 0; h < NH; h++) {
                        const unsigned m = __reduce_max_sync(0xffffffffu, __float_as_uint(fabsf(qv[h])));
                        if (lane == 0) s_red[warp][h] = __uint_as_float(m);
                    }
                    wg_sync();
#pragma unroll
                    for (int h = 0; h < NH; h++) {
                        const float m = fmaxf(fmaxf(s_red[0][h], s_red[1][h]), fmaxf(s_red[2][h], s_red[3][h]));
                        int e = static_cast<int>(__float_as_uint(m) >> 23) - 127 - 9;   // m in [2^(e+9), 2^(e+10))
                        e = max(-110, min(110, e));
                        fh[h] = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
                        qv[h] *= __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
                    }
                    wg_sync();
                } else {
#pragma unroll
                    for (int h = 0; h < NH; h++) fh[h] = 1.f;
                }
#pragma unroll
                for (int h = 0; h < NH; h++) {
                    uint16_t t[TERMS];
                    split<BF>(qv[h], t);
#pragma unroll
                    for (int i = 0; i < TERMS; i++) *reinterpret_cast<uint16_t *>(sQ + b_off(NB, i * NH + h, tid)) = t[i];
                }
                fence_async();
                mbar_arrive(&bars.qfull);
            }
            float m[NH], l[NH];
#pragma unroll
            for (int h = 0; h < NH; h++) {
                m[h] = -INFINITY;
                l[h] = 0.f;
            }
            const int ntp = wk.t1 - wk.t0;
            int row = (s.tile0 + wk.t0) * kTile + tid;
            auto page_ok = [&](int r) {
                return r >= s.first && r < s.n &&
                       static_cast<unsigned>(__ldg(table + (r >> kv.page_shift))) < static_cast<unsigned>(kv.n_pages);
            };
            bool on = page_ok(row);
            for (int t = 0; t < ntp; t++, q++, row += kTile) {
                const bool on_next = t + 1 < ntp && page_ok(row + kTile);
                wait(&bars.sfull[q & 1], static_cast<uint32_t>((q >> 1) & 1));
                __syncwarp();
                fence_after();
                float sv[NB];
                ld_cols<NB>(tmem + (q & 1) * kColS + lane_base, sv);
                float x[NH];
                bool up = false;
#pragma unroll
                for (int h = 0; h < NH; h++) {
                    float y = sv[h] + sv[NH + h];
                    if constexpr (TERMS == 3) y = sv[h] + (sv[NH + h] + sv[2 * NH + h]);
                    x[h] = on ? y * fh[h] : -INFINITY;
                    up |= x[h] > m[h] + kSlack;
                }
                if (a.acc_out && on) {
                    float *sc = a.scores + ((static_cast<long long>(wk.b) * kv.n_kv + j) * max_rows + row) * a.gqa + g0;
                    if (ng == NH && (a.gqa & 3) == 0) {
#pragma unroll
                        for (int h = 0; h < NH; h += 4) *reinterpret_cast<float4 *>(sc + h) = make_float4(x[h], x[h + 1], x[h + 2], x[h + 3]);
                    } else {
#pragma unroll
                        for (int h = 0; h < NH; h++)
                            if (h < ng) sc[h] = x[h];
                    }
                }
                if (wg_any(up)) {
                    // new maxima over the tile's rows; what was summed against the old ones is rescaled
#pragma unroll
                    for (int h = 0; h < NH; h++) {
                        float v = x[h];
#pragma unroll
                        for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
                        if (lane == 0) s_red[warp][h] = v;
                    }
                    wg_sync();
                    float f[NH];
#pragma unroll
                    for (int h = 0; h < NH; h++) {
                        const float v = fmaxf(m[h], fmaxf(fmaxf(s_red[0][h], s_red[1][h]), fmaxf(s_red[2][h], s_red[3][h])));
                        f[h] = m[h] > -INFINITY ? ex2(m[h] - v) : 0.f;
                        l[h] *= f[h];
                        m[h] = v;
                    }
                    wg_sync();   // s_red is free again
                    if (t > 0) {
                        wait(&bars.odone, static_cast<uint32_t>((q - 1) & 1));
                        __syncwarp();
                        fence_after();
                        float ov[NB];
                        ld_cols<NB>(tmem + kColO + lane_base, ov);
#pragma unroll
                        for (int h = 0; h < NH; h++)
#pragma unroll
                            for (int i = 0; i < TERMS; i++) ov[i * NH + h] *= f[h];
#pragma unroll
                        for (int c = 0; c < NB; c += 8) st8(tmem + kColO + lane_base + c, ov + c);
                        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    }
                }
                if (t > 0) wait(&bars.odone, static_cast<uint32_t>((q - 1) & 1));   // P is free
                __syncwarp();
#pragma unroll
                for (int h = 0; h < NH; h++) {
                    const float p = on ? ex2(x[h] - (m[h] > -INFINITY ? m[h] : 0.f)) : 0.f;
                    l[h] += p;
                    uint16_t tt[TERMS];
                    split<BF>(BF ? p : p * 128.f, tt);
#pragma unroll
                    for (int i = 0; i < TERMS; i++) *reinterpret_cast<uint16_t *>(sP + b_off(NB, i * NH + h, tid)) = tt[i];
                }
                if (!on) {
                    // 0 x (whatever lies in a row that is not seen) has to be 0
                    const int st = q % kStages;
                    wait(&bars.vfull[st], static_cast<uint32_t>((q / kStages) & 1));
                    const uint4 z = make_uint4(0, 0, 0, 0);
                    uint8_t *vr = sV + st * kSlotBytes + tid * 128;
#pragma unroll
                    for (int c = 0; c < 8; c++) {
                        *reinterpret_cast<uint4 *>(vr + 16 * c) = z;
                        *reinterpret_cast<uint4 *>(vr + kHalfBytes + 16 * c) = z;
                    }
                }
                __syncwarp();
                fence_async();
                fence_before();
                mbar_arrive(&bars.pfull);
                on = on_next;
            }
            wait(&bars.odone, static_cast<uint32_t>((q - 1) & 1));
            __syncwarp();
            fence_after();
            // ---------------- the portion's end: thread = element of head_dim
            float ov[NB], o[NH];
            ld_cols<NB>(tmem + kColO + lane_base, ov);
#pragma unroll
            for (int h = 0; h < NH; h++) {
                o[h] = TERMS == 3 ? ov[h] + (ov[NH + h] + ov[(TERMS - 1) * NH + h]) : ov[h] + ov[NH + h];
                if constexpr (!BF) o[h] *= 0x1p-7f;
                float v = l[h];
#pragma unroll
                for (int k = 16; k; k >>= 1) v += __shfl_xor_sync(0xffffffffu, v, k);
                if (lane == 0) s_red[warp][h] = v;
            }
            fence_before();
            wg_sync();
            float L[NH];
#pragma unroll
            for (int h = 0; h < NH; h++) L[h] = (s_red[0][h] + s_red[1][h]) + (s_red[2][h] + s_red[3][h]);
            // whole segment: out; else a part of it
            const long long seg_at = wk.at - wk.t1;              // the segment's first tile in the list
            const long long own0 = ((seg_at + 1) * G - 1) / T, own1 = ((seg_at + wk.nt) * G - 1) / T;
            if (own0 == own1) {
#pragma unroll
                for (int h = 0; h < NH; h++)
                    if (h < ng) {
                        if (tid < kv.hd) a.out[(h0 + h) * kv.hd + tid] = L[h] > 0.f ? o[h] / L[h] : 0.f;
                        if (tid == h) {
                            if (a.lse) a.lse[h0 + h] = L[h] > 0.f ? m[h] * 0.6931471805599453f + logf(L[h]) : -INFINITY;
                            if (a.acc_out) {
                                a.ml[2 * (h0 + h)] = m[h];
                                a.ml[2 * (h0 + h) + 1] = L[h];
                            }
                        }
                    }
                wg_sync();   // s_red
                continue;
            }
            const int slot = 2 * static_cast<int>(blockIdx.x) + (wk.t0 == 0 ? 1 : 0);
            float *part = a.part + static_cast<long long>(slot) * kAttendPart;
#pragma unroll
            for (int h = 0; h < NH; h++) {
                part[h * 128 + tid] = o[h];
                if (tid == h) {
                    part[NH * 128 + h] = m[h];
                    part[NH * 128 + NH + h] = L[h];
                }
            }
            wg_sync();
            if (tid == 0) {
                __threadfence();
                unsigned *cnt = a.cnt + static_cast<long long>(wk.b) * segs + wk.seg;
                s_last = atomicAdd(cnt, 1u) == static_cast<unsigned>(own1 - own0);
                if (s_last) *cnt = 0;   // for the next call
                __threadfence();
            }
            wg_sync();
            if (s_last) {
                // part i is of CTA own0 + i: slot 2 own0 + 1, then 2 (own0 + i)
                const int np = static_cast<int>(own1 - own0) + 1;
                auto part_of = [&](int i) {
                    return a.part + (2 * (own0 + i) + (i == 0 ? 1 : 0)) * kAttendPart;
                };
                float *wgt = reinterpret_cast<float *>(sQ);   // [np][NH]: Q and P are not in use
                for (int i = tid; i < np * NH; i += 128) wgt[i] = __ldcg(part_of(i / NH) + NH * 128 + i % NH);
                wg_sync();
                float M[NH];
#pragma unroll
                for (int h = 0; h < NH; h++) M[h] = -INFINITY;
                for (int i = 0; i < np; i++)
#pragma unroll
                    for (int h = 0; h < NH; h++) M[h] = fmaxf(M[h], wgt[i * NH + h]);
                wg_sync();
                if (tid < NH) {
#pragma unroll
                    for (int h = 0; h < NH; h++)
                        if (tid == h) s_f[h] = M[h];
                }
                wg_sync();
                for (int i = tid; i < np * NH; i += 128) {
                    const float mi = wgt[i], MM = s_f[i % NH];
                    wgt[i] = mi > -INFINITY ? ex2(mi - MM) : 0.f;
                }
                wg_sync();
                float acc[NH], Ls[NH];
#pragma unroll
                for (int h = 0; h < NH; h++) {
                    acc[h] = 0.f;
                    Ls[h] = 0.f;
                }
#pragma unroll 4
                for (int i = 0; i < np; i++) {
                    const float *pp = part_of(i);
#pragma unroll
                    for (int h = 0; h < NH; h++) {
                        const float f = wgt[i * NH + h];
                        acc[h] += f * __ldcg(pp + h * 128 + tid);
                        Ls[h] += f * __ldcg(pp + NH * 128 + NH + h);
                    }
                }
#pragma unroll
                for (int h = 0; h < NH; h++)
                    if (h < ng) {
                        if (tid < kv.hd) a.out[(h0 + h) * kv.hd + tid] = Ls[h] > 0.f ? acc[h] / Ls[h] : 0.f;
                        if (tid == h) {
                            if (a.lse) a.lse[h0 + h] = Ls[h] > 0.f ? M[h] * 0.6931471805599453f + logf(Ls[h]) : -INFINITY;
                            if (a.acc_out) {
                                a.ml[2 * (h0 + h)] = M[h];
                                a.ml[2 * (h0 + h) + 1] = Ls[h];
                            }
                        }
                    }
                wg_sync();   // the weights' place is Q's again
            }
        }
    }
    __syncthreads();
    if (warp == kWarpMma)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
}

template <bool BF, int NH>
cudaError_t launch(const PagedAttendArgs &a, const CUtensorMap &mk, const CUtensorMap &mv, int grid, cudaStream_t st) {
    constexpr int smem = Cfg<BF, NH>::smem;
    static_assert(smem <= 227 * 1024 - 8 * 1024, "shared memory");
    const cudaError_t e = cudaFuncSetAttribute(k_attend_tc<BF, NH>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    return launch_pdl(k_attend_tc<BF, NH>, dim3(grid), dim3(kThreads), smem, st, a, mk, mv);
}

}  // namespace

cudaError_t launch_attend_tc(const PagedAttendArgs &a, const CUtensorMap &mk, const CUtensorMap &mv, int sms, cudaStream_t st) {
    const int nh = a.gqa <= 8 ? 8 : 16, groups = (a.gqa + nh - 1) / nh;
    // no more CTAs than tiles there can be
    const long long tiles = static_cast<long long>(a.kv.n_seqs) * a.kv.n_kv * groups *
                            (((static_cast<long long>(a.kv.max_pages) << a.kv.page_shift) + kTile - 1) / kTile);
    const int grid = static_cast<int>(tiles < sms ? tiles : sms);
    if (a.kv.dtype == STYX_BF16) return nh == 8 ? launch<true, 8>(a, mk, mv, grid, st) : launch<true, 16>(a, mk, mv, grid, st);
    return nh == 8 ? launch<false, 8>(a, mk, mv, grid, st) : launch<false, 16>(a, mk, mv, grid, st);
}

}  // namespace styx
