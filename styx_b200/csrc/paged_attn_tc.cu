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
// written out where it is the whole segment, else to the workspace, from
// where k_attend_finish adds the portions up in order.
// (Joining inside this kernel, by the CTA that finishes a segment last, kept
// four of 148 SMs 12 us longer than the rest at one sequence of 131071 rows.)
//
// Roles, linked by mbarriers with bounded waits: two softmax warpgroups take
// alternate tiles (thread = row of the tile), each with its own score buffer,
// maxima, sums, P and accumulator, so that one's chain scores -> exponentials
// -> P -> product overlaps the other's; they are added up at the portion's
// end (thread = element of head_dim).  One warp copies K, one copies V, one
// issues S, one O.  K and V share one ring of 16 KB slots (half the columns
// of a K tile, half the rows of a V tile), 11 or 12 of them, filled in the
// order K0 K1 V0 K2 V1 K3 ... in which they are used, so the whole 176 to 192
// KB are in flight for whichever is needed next.  The maximum a row is measured
// against moves only when a score passes it by 2^8, so the accumulator is
// rescaled rarely and no tile waits for an exact running maximum; sums and
// exponentials are unaffected by which one is used.
#include <cuda_runtime.h>

#include <cstdint>

#include "paged_split.cuh"

namespace styx {
namespace {

constexpr int kHalfBytes = kTile * 128;    // 64 columns of a tile: 128-byte rows
constexpr int kSlotBytes = kHalfBytes;     // K: 128 rows x 64 columns; V: 2 x (64 rows x 64 columns)
constexpr int kThreads = 384;
constexpr int kWarpK = 8, kWarpV = 9, kWarpS = 10, kWarpO = 11;
constexpr uint32_t kTmemCols = 256, kColS = 0, kColO = 128, kColStep = 64;   // two score buffers, two accumulators
constexpr float kSlack = 8.f;              // log2 units a score may pass the maximum by

template <bool BF, int NH>
struct Cfg {
    static constexpr int terms = BF ? 3 : 2;
    static constexpr int nb = (terms * NH + 15) / 16 * 16;   // N of the products (M 128: multiples of 16)
    static constexpr int q_bytes = 2 * nb * 128, p_bytes = 2 * nb * 128;
    static constexpr int slots = NH == 8 ? 12 : 11;                  // what 227 KB hold
    static constexpr int qn_bytes = NH * 128 * 4;                    // the next portion's q
    static constexpr int smem = slots * kSlotBytes + q_bytes + 2 * p_bytes + qn_bytes + 1024;
    // term of a small p keeps its bits; bf16 has f32's range
};

// ------------------------------------------------------------ tensor-core helpers
// Shared-memory operand descriptors (version 1, 128-byte swizzle).  The high
// word is the same for all: 1024 bytes between groups of 8 rows (K-major) or
// of 8 along K (M-major).  The low word is address / 16, and for M-major the
// bytes / 16 between blocks of 64 along M: advancing is an addition.
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t lbo) { return (addr >> 4) | ((lbo >> 4) << 16); }
// f32 accumulator, A and B both f16 or both bf16, M 128; a_mn: A is M-major
constexpr uint32_t idesc(bool bf, int n, bool a_mn) {
    return (1u << 4) | (bf ? (1u << 7) | (1u << 10) : 0u) | (a_mn ? 1u << 15 : 0u) |
           (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(kTile >> 4) << 24);
}
__device__ __forceinline__ void mma(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t id, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "mov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}\n" ::"r"(d),
        "r"(a_lo), "r"(b_lo), "r"(id), "r"(acc), "n"(kDescHi));
}
__device__ __forceinline__ bool elect() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
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
// the loads above are done; no use of their values moves up across this
template <int N>
__device__ __forceinline__ void ld_done(float (&v)[N]) {
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
// barriers of one softmax warpgroup (0 or 1), and of both
__device__ __forceinline__ void wg_sync(int wg) { asm volatile("bar.sync %0, 128;" ::"r"(1 + wg) : "memory"); }
__device__ __forceinline__ void both_sync() { asm volatile("bar.sync 3, 256;" ::: "memory"); }
__device__ __forceinline__ void read_arrive() { asm volatile("bar.arrive 4, 256;" ::: "memory"); }
__device__ __forceinline__ void read_sync() { asm volatile("bar.sync 4, 256;" ::: "memory"); }
__device__ __forceinline__ bool wg_any(int wg, bool v) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\t"
        "barrier.cta.red.or.pred q, %2, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r)
        : "r"(static_cast<uint32_t>(v)), "r"(1 + wg)
        : "memory");
    return r != 0;
}
__device__ __forceinline__ float warp_max(float v) {   // NaN only where every lane has it
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}
// v as a sum of terms of the cache's type, largest first.  bf16: the f32's 24
// significant bits cut into 8 + 8 + 8, exactly; f16: rounded to 11, the rest
// rounded to 11.
template <bool BF>
__device__ __forceinline__ void split(float v, uint16_t (&t)[BF ? 3 : 2]) {
    if constexpr (BF) {
        const uint32_t a = __float_as_uint(v);
        const uint32_t b = __float_as_uint(v - __uint_as_float(a & 0xFFFF0000u));
        const uint32_t c = __float_as_uint(__uint_as_float(b) - __uint_as_float(b & 0xFFFF0000u));
        t[0] = static_cast<uint16_t>(a >> 16);
        t[1] = static_cast<uint16_t>(b >> 16);
        t[2] = static_cast<uint16_t>(c >> 16);
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
    uint64_t full[12], empty[12];
    uint64_t sfull[2], pfull[2], odone[2], qfull, drain[2];
};

// Position of a portion's copies in its list (K0 K1 V0 K2 V1 ... of nt tiles,
// kh slots for a K tile, 2 for a V tile)
__device__ __forceinline__ int pos_k(int t, int kh) { return kh * t + 2 * max(0, t - 1); }
__device__ __forceinline__ int pos_v(int t, int nt, int kh) { return kh * min(t + 2, nt) + 2 * t; }

template <bool BF, int NH>
__global__ void __launch_bounds__(kThreads, 1)
    k_attend_tc(PagedAttendArgs a, const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv) {
    using C = Cfg<BF, NH>;
    constexpr int NB = C::nb, TERMS = C::terms;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *sm = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
    uint8_t *ring = sm, *sQ = ring + C::slots * kSlotBytes, *sP = sQ + C::q_bytes;
    float *sQn = reinterpret_cast<float *>(sP + 2 * C::p_bytes);
    __shared__ Bars bars;
    __shared__ uint32_t s_tmem;
    __shared__ Share<kThreads> share;
    __shared__ int s_abort;
    __shared__ float s_red[8][16], s_l[8][16], s_ml[2][16], s_f[16];
    const PagedKv &kv = a.kv;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const int groups = (a.gqa + NH - 1) / NH, segs = kv.n_kv * groups;

    pdl_trigger();
    if (tid == 32 * kWarpK) asm volatile("prefetch.tensormap [%0];" ::"l"(&mk));
    if (tid == 32 * kWarpV) asm volatile("prefetch.tensormap [%0];" ::"l"(&mv));
    if (tid == 0) {
        for (int i = 0; i < C::slots; i++) {
            mbar_init(&bars.full[i], 1);
            mbar_init(&bars.empty[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&bars.sfull[i], 1);
            mbar_init(&bars.pfull[i], 128);
            mbar_init(&bars.odone[i], 1);
        }
        mbar_init(&bars.qfull, 128);
        mbar_init(&bars.drain[0], 1);
        mbar_init(&bars.drain[1], 1);
        fence_mbar_init();
        s_abort = 0;
    }
    if (warp == kWarpO) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&s_tmem)),
                     "r"(kTmemCols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    pdl_wait();

    long long T, G;
    Walk wk;
    share_of<kThreads>(a, segs, share, wk, T, G);
    const uint32_t tmem = s_tmem;
    const int kh = kv.hd > 64 ? 2 : 1;   // K slots of a tile

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
        // (V: min(page, 64) rows).  Lane = box; a slot's boxes are of eight
        // or fewer neighbouring lanes.
        const bool isv = warp == kWarpV;
        const CUtensorMap *map = isv ? &mv : &mk;
        const int rb_shift = min(kv.page_shift, isv ? 6 : 7), rows = 1 << rb_shift;
        const int halves = kh, nbox = kTile >> rb_shift;      // boxes along the rows (<= 8) and the columns
        // K: slot = column half, boxes along the rows; V: slot = row half, boxes (rows of it) x column halves
        const int n_slots = isv ? 2 : kh, per = isv ? nbox / 2 * halves : nbox;
        const int sl = lane / per, in = lane - sl * per;      // this lane's slot and box in it
        const int pi = isv ? sl * (nbox / 2) + in / halves : in, half = isv ? in % halves : sl;
        const bool mine = lane < n_slots * per;
        const int dst = isv ? half * (64 * 128) + (((in / halves) << rb_shift) * 128) : (pi << rb_shift) * 128;
        const unsigned slot_lanes = mine ? ((1u << per) - 1u) << (sl * per) : 0u;
        // a tile's box of this lane: the page's id (loaded one tile ahead) and the row in the page
        struct Box {
            bool on;
            int page, y;
        };
        bool more = wk.next(a, segs);
        int t = wk.t0, base = 0, nt = wk.t1 - wk.t0, i = 0;   // the portion's first position, its tiles, the tile in it
        auto fetch = [&]() {
            Box x{false, 0, 0};
            if (!more) return x;
            const Seq s(a, wk.b, false);
            const int r0 = (s.tile0 + t) * kTile + (pi << rb_shift);
            x.on = mine && r0 < s.n && r0 + rows > s.first;
            if (x.on) x.page = __ldg(kv.table + static_cast<long long>(wk.b) * kv.table_stride + (r0 >> kv.page_shift));
            x.y = ((wk.seg / groups) << kv.page_shift) + (r0 & ((1 << kv.page_shift) - 1));
            return x;
        };
        Box nxt = fetch();
        while (more) {
            Box x = nxt;
            const int first = base + (isv ? pos_v(i, nt, kh) : pos_k(i, kh));
            i++;
            if (++t == wk.t1) {
                base += nt * (kh + 2);
                more = wk.next(a, segs);
                t = wk.t0;
                nt = wk.t1 - wk.t0;
                i = 0;
            }
            nxt = fetch();
            if (x.on && static_cast<unsigned>(x.page) >= static_cast<unsigned>(kv.n_pages)) {
                if (!isv) atomicExch(kv.err, kErrBadPos);
                x.on = false;
            }
            const unsigned on = __ballot_sync(0xffffffffu, x.on);
            // the slots in order: a slot is armed, then its lanes copy
            bool live = true;
            for (int k = 0; k < n_slots; k++) {
                const int p = first + k, st = p % C::slots, use = p / C::slots;
                if (use > 0 && !__all_sync(0xffffffffu, wait(&bars.empty[st], static_cast<uint32_t>((use - 1) & 1)))) {
                    live = false;
                    break;
                }
                const unsigned lanes = __shfl_sync(0xffffffffu, slot_lanes, k * per);
                if (lane == 0)
                    mbar_arrive_expect_tx(&bars.full[st], __popc(on & lanes) * static_cast<uint32_t>(rows) * 128u);
                __syncwarp();
                if (x.on && sl == k) tma3(ring + st * kSlotBytes + dst, map, half * 64, x.y, x.page, &bars.full[st]);
            }
            if (!live) break;
        }
        // Every copy is waited for by the products that read it.  Where a wait gave up, nothing of this warp's may still
        // be landing when the CTA ends: copies take microseconds, a millisecond is given to them.
        if (*reinterpret_cast<volatile int *>(&s_abort))
            for (const long long c0 = clock64(); clock64() - c0 < 2000000;) {
            }
    } else if (warp == kWarpS) {
        // ---------------- S = K Q^T.  The warp walks together (what an MMA is
        // given stays in uniform registers), one lane issues.
        constexpr uint32_t id = idesc(BF, NB, false);
        const bool leader = elect();
        const int ksteps = (kv.hd + 15) / 16;
        const uint32_t dK = desc_lo(smem_addr(ring), 16), dQ = desc_lo(smem_addr(sQ), 16);
        int q = 0, portion = 0, base = 0;   // tile number, portion, its first slot position
        bool live = true;
        while (live && wk.next(a, segs)) {
            const int nt = wk.t1 - wk.t0;
            int st = base % C::slots;
            uint32_t ph = static_cast<uint32_t>(base / C::slots) & 1;
            live = wait(&bars.qfull, static_cast<uint32_t>(portion & 1));
            for (int t = 0; t < nt; t++, q++) {
                // the buffer's earlier scores (tile q - 2) have been read
                if (q > 1) live &= wait(&bars.pfull[q & 1], static_cast<uint32_t>((q >> 1) + 1) & 1);
                const int s1 = st + 1 == C::slots ? 0 : st + 1;
                live &= wait(&bars.full[st], ph);
                if (kh == 2) live &= wait(&bars.full[s1], st + 1 == C::slots ? ph ^ 1 : ph);
                fence_after();
                if (leader) {
                    const uint32_t d = tmem + kColS + (q & 1) * kColStep;
#pragma unroll
                    for (int k = 0; k < 8; k++)
                        if (k < ksteps)
                            mma(d, dK + static_cast<uint32_t>(k < 4 ? st : s1) * (kSlotBytes / 16) + (k & 3) * 2,
                                dQ + (k >> 2) * (NB * 128 / 16) + (k & 3) * 2, id, k > 0);
                    commit(&bars.sfull[q & 1]);
                    commit(&bars.empty[st]);
                    if (kh == 2) commit(&bars.empty[s1]);
                }
                live = __all_sync(0xffffffffu, live);
                if (!live) break;
                st += t == 0 ? kh : kh + 2;   // K0 K1 V0 K2 V1 ...
                if (st >= C::slots) {
                    st -= C::slots;
                    ph ^= 1;
                }
            }
            base += nt * (kh + 2);
            portion++;
        }
        if (leader) {   // every product issued here has completed before TMEM is freed
            commit(&bars.drain[0]);
            mbar_wait(&bars.drain[0], 0u, nullptr, 0);
        }
        __syncwarp();
    } else if (warp == kWarpO) {
        // ---------------- O^T += V^T P^T
        constexpr uint32_t id = idesc(BF, NB, true);
        const bool leader = elect();
        const uint32_t dV = desc_lo(smem_addr(ring), 64 * 128), dP = desc_lo(smem_addr(sP), 16);
        int q = 0, base = 0;
        bool live = true;
        while (live && wk.next(a, segs)) {
            const int nt = wk.t1 - wk.t0, p0 = base + pos_v(0, nt, kh);
            int st = p0 % C::slots;
            uint32_t ph = static_cast<uint32_t>(p0 / C::slots) & 1;
            for (int t = 0; t < nt; t++, q++) {
                const int wg = q & 1, s1 = st + 1 == C::slots ? 0 : st + 1;
                live &= wait(&bars.full[st], ph);
                live &= wait(&bars.full[s1], st + 1 == C::slots ? ph ^ 1 : ph);
                live &= wait(&bars.pfull[wg], static_cast<uint32_t>((q >> 1) & 1));
                fence_after();
                if (leader) {
                    const uint32_t d = tmem + kColO + wg * kColStep, dp = dP + static_cast<uint32_t>(wg) * (C::p_bytes / 16);
#pragma unroll
                    for (int k = 0; k < 8; k++)
                        mma(d, dV + static_cast<uint32_t>(k < 4 ? st : s1) * (kSlotBytes / 16) + (k & 3) * (2048 / 16),
                            dp + (k >> 2) * (NB * 128 / 16) + (k & 3) * 2, id, t > 1 || k > 0);
                    commit(&bars.odone[wg]);
                    commit(&bars.empty[st]);
                    commit(&bars.empty[s1]);
                }
                live = __all_sync(0xffffffffu, live);
                if (!live) break;
                st += t + 2 < nt ? kh + 2 : 2;
                if (st >= C::slots) {
                    st -= C::slots;
                    ph ^= 1;
                }
            }
            base += nt * (kh + 2);
        }
        if (leader) {
            commit(&bars.drain[1]);
            mbar_wait(&bars.drain[1], 0u, nullptr, 0);
        }
        __syncwarp();
    } else {
        // ---------------- softmax: thread = row of the tile.  A wait that gave
        // up is not looked at here: every thread goes on to the end, so the
        // warps stay together at their barriers (later waits return at once,
        // the results are void and the error word says so).
        const int wg = warp >> 2, tg = tid & 127;
        const uint32_t lane_base = static_cast<uint32_t>(32 * (warp & 3)) << 16;
        const uint32_t colS = tmem + kColS + wg * kColStep + lane_base, colO = tmem + kColO + wg * kColStep + lane_base;
        uint8_t *myP = sP + wg * C::p_bytes;
        const float l2 = a.scale * 1.4426950408889634f;   // scores in units of log2
        const long long max_rows = static_cast<long long>(kv.max_pages) << kv.page_shift;
        int q = 0, portion = 0, base = 0;                  // the portion's first tile, its number, its first slot position
        // q of a portion into shared memory: every thread the elements that it will read itself
        auto stage_q = [&](const Walk &w) {
            const int j = w.seg / groups, g0 = (w.seg - j * groups) * NH;
            const float *qp = a.q + (static_cast<long long>(w.b) * a.n_heads + j * a.gqa + g0) * kv.hd + tg;
#pragma unroll
            for (int h = 0; h < NH; h++)
                if (h < a.gqa - g0 && tg < kv.hd)
                    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_addr(sQn + h * 128 + tg)),
                                 "l"(qp + h * kv.hd)
                                 : "memory");
        };
        while (wk.next(a, segs)) {
            const Seq s(a, wk.b, false);
            const int j = wk.seg / groups, g0 = (wk.seg - j * groups) * NH, ng = min(NH, a.gqa - g0);
            const long long h0 = static_cast<long long>(wk.b) * a.n_heads + j * a.gqa + g0;
            const int32_t *table = kv.table + static_cast<long long>(wk.b) * kv.table_stride;
            if (wg == 1) {
                // Q, by the second warpgroup, so that the next portion starts while the first still writes the last
                // one's result.  Thread = element.  f16 has few exponents: every head's largest |q| is brought to
                // [2^9, 2^10), and s_f says what a column of S is in units of its terms.
                float qv[NH];
                if (portion == 0) stage_q(wk);
                asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll
                for (int h = 0; h < NH; h++) qv[h] = h < ng && tg < kv.hd ? sQn[h * 128 + tg] * l2 : 0.f;
                if constexpr (!BF) {
#pragma unroll
                    for (int h = 0; h < NH; h++) {
                        const unsigned mx = __reduce_max_sync(0xffffffffu, __float_as_uint(fabsf(qv[h])));
                        if (lane == 0) s_red[warp][h] = __uint_as_float(mx);
                    }
                    wg_sync(1);
#pragma unroll
                    for (int h = 0; h < NH; h++) {
                        const float *r = &s_red[4][h];
                        const float mx = fmaxf(fmaxf(r[0], r[16]), fmaxf(r[32], r[48]));
                        int e = static_cast<int>(__float_as_uint(mx) >> 23) - 127 - 9;
                        e = max(-110, min(110, e));
                        if (tg == 0) s_f[h] = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
                        qv[h] *= __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
                    }
                }
#pragma unroll
                for (int h = 0; h < NH; h++) {
                    uint16_t t[TERMS];
                    split<BF>(qv[h], t);
#pragma unroll
                    for (int i = 0; i < TERMS; i++) *reinterpret_cast<uint16_t *>(sQ + b_off(NB, i * NH + h, tg)) = t[i];
                }
                fence_async();
                mbar_arrive(&bars.qfull);
                Walk ahead = wk;   // the next portion's q is on its way while this one runs
                if (ahead.next(a, segs)) stage_q(ahead);
                if (portion > 0) read_sync();   // the first warpgroup has read what lies in this one's P
            }
            if constexpr (!BF) {
                wait(&bars.qfull, static_cast<uint32_t>(portion & 1));   // s_f
                __syncwarp();
            }
            portion++;
            float fh[NH], m[NH], l[NH];
#pragma unroll
            for (int h = 0; h < NH; h++) {
                fh[h] = BF ? 1.f : s_f[h];
                m[h] = kNone;
                l[h] = 0.f;
            }
            const int ntp = wk.t1 - wk.t0, t_first = (q ^ wg) & 1;   // this warpgroup's tiles: t_first, t_first + 2, ...
            int row = (s.tile0 + wk.t0 + t_first) * kTile + tg;
            auto page_of = [&](int r) { return r >= s.first && r < s.n ? __ldg(table + (r >> kv.page_shift)) : -1; };
            int page = t_first < ntp ? page_of(row) : -1;
            for (int t = t_first; t < ntp; t += 2, row += 2 * kTile) {
                const int qt = q + t;
                const uint32_t par = static_cast<uint32_t>((qt >> 1) & 1);
                const bool on = static_cast<unsigned>(page) < static_cast<unsigned>(kv.n_pages);
                page = t + 2 < ntp ? page_of(row + 2 * kTile) : -1;   // loaded one tile ahead
                wait(&bars.sfull[wg], par);
                __syncwarp();
                fence_after();
                float x[NH];
                bool up = false;
#pragma unroll
                for (int hb = 0; hb < NH; hb += 8) {   // by eight heads: fewer registers at once
                    float sv[TERMS * 8];
#pragma unroll
                    for (int i = 0; i < TERMS; i++) ld8(colS + i * NH + hb, sv + 8 * i);
                    ld_done(sv);
#pragma unroll
                    for (int h = 0; h < 8; h++) {
                        const float y = TERMS == 3 ? sv[h] + (sv[8 + h] + sv[(TERMS - 1) * 8 + h]) : sv[h] + sv[8 + h];
                        x[hb + h] = on ? (BF ? y : y * fh[hb + h]) : -INFINITY;
                        up |= x[hb + h] > m[hb + h] + kSlack;
                    }
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
                if (wg_any(wg, up)) {
                    // new maxima over the tile's rows; what was summed against the old ones is rescaled
#pragma unroll
                    for (int h = 0; h < NH; h++) {
                        const float v = warp_max(x[h]);
                        if (lane == 0) s_red[warp][h] = v;
                    }
                    wg_sync(wg);
                    if (t > 1) wait(&bars.odone[wg], par ^ 1u);
                    __syncwarp();
                    fence_after();
#pragma unroll
                    for (int hb = 0; hb < NH; hb += 8) {
                        float f[8];
#pragma unroll
                        for (int h = 0; h < 8; h++) {
                            const float *r = &s_red[4 * wg][hb + h];
                            const float v = fmaxf(m[hb + h], fmaxf(fmaxf(r[0], r[16]), fmaxf(r[32], r[48])));
                            f[h] = ex2(m[hb + h] - v);
                            l[hb + h] *= f[h];
                            m[hb + h] = v;
                        }
                        if (t > 1) {
                            float ov[TERMS * 8];
#pragma unroll
                            for (int i = 0; i < TERMS; i++) ld8(colO + i * NH + hb, ov + 8 * i);
                            ld_done(ov);
#pragma unroll
                            for (int h = 0; h < 8; h++)
#pragma unroll
                                for (int i = 0; i < TERMS; i++) ov[8 * i + h] *= f[h];
#pragma unroll
                            for (int i = 0; i < TERMS; i++) st8(colO + i * NH + hb, ov + 8 * i);
                        }
                    }
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    wg_sync(wg);   // s_red is free again
                }
                if (t > 1) wait(&bars.odone[wg], par ^ 1u);   // P is free
                __syncwarp();
#pragma unroll
                for (int h = 0; h < NH; h++) {
                    const float p = on ? ex2(x[h] - m[h]) : 0.f;
                    l[h] += p;
                    uint16_t tt[TERMS];
                    // f16: p up to 2^8 is carried as p * 2^7, so that the second term of a small p keeps its bits
                    split<BF>(BF ? p : p * 128.f, tt);
#pragma unroll
                    for (int i = 0; i < TERMS; i++) *reinterpret_cast<uint16_t *>(myP + b_off(NB, i * NH + h, tg)) = tt[i];
                }
                if (!on) {
                    // 0 x (whatever lies in a row that is not seen) has to be 0
                    const int p = base + pos_v(t, ntp, kh) + (tg >> 6), st = p % C::slots;
                    wait(&bars.full[st], static_cast<uint32_t>((p / C::slots) & 1));
                    const uint4 z = make_uint4(0, 0, 0, 0);
                    uint8_t *vr = ring + st * kSlotBytes + (tg & 63) * 128;
#pragma unroll
                    for (int c = 0; c < 8; c++) {
                        *reinterpret_cast<uint4 *>(vr + 16 * c) = z;
                        *reinterpret_cast<uint4 *>(vr + 64 * 128 + 16 * c) = z;
                    }
                }
                __syncwarp();
                fence_async();
                fence_before();
                mbar_arrive(&bars.pfull[wg]);
            }
            // ---------------- the portion's end: thread = element of head_dim
            const bool any = t_first < ntp;
            if (any) wait(&bars.odone[wg], static_cast<uint32_t>(((q + ((ntp - 1 - t_first) & ~1) + t_first) >> 1) & 1));
            __syncwarp();
            fence_after();
            q += ntp;
            base += ntp * (kh + 2);
            float o[NH];
#pragma unroll
            for (int hb = 0; hb < NH; hb += 8) {
                float ov[TERMS * 8];
                if (any) {
#pragma unroll
                    for (int i = 0; i < TERMS; i++) ld8(colO + i * NH + hb, ov + 8 * i);
                    ld_done(ov);
                }
#pragma unroll
                for (int h = 0; h < 8; h++) {
                    const float y = TERMS == 3 ? ov[h] + (ov[8 + h] + ov[(TERMS - 1) * 8 + h]) : ov[h] + ov[8 + h];
                    o[hb + h] = any ? (BF ? y : y * 0x1p-7f) : 0.f;
                }
            }
            fence_before();
#pragma unroll
            for (int h = 0; h < NH; h++) {
                float v = l[h];
#pragma unroll
                for (int k = 16; k; k >>= 1) v += __shfl_xor_sync(0xffffffffu, v, k);
                if (lane == 0) s_l[warp][h] = v;
            }
            // the second warpgroup's share goes through its P
            float *ex = reinterpret_cast<float *>(sP + C::p_bytes);
            if (wg == 1) {
#pragma unroll
                for (int h = 0; h < NH; h++) {
                    ex[h * 128 + tg] = o[h];
                    if (tg == h) s_ml[1][h] = m[h];
                }
            }
            both_sync();
            if (wg == 1) continue;
            float L[NH];
#pragma unroll
            for (int h = 0; h < NH; h++) {
                const float *r = &s_l[0][h];
                const float L0 = (r[0] + r[16]) + (r[32] + r[48]), L1 = (r[64] + r[80]) + (r[96] + r[112]);
                const float m1 = s_ml[1][h], M = fmaxf(m[h], m1), f0 = ex2(m[h] - M), f1 = ex2(m1 - M);
                o[h] = o[h] * f0 + ex[h * 128 + tg] * f1;
                L[h] = L0 * f0 + L1 * f1;
                m[h] = M;
            }
            read_arrive();
            auto write_out = [&](const float (&ov)[NH], const float (&mv)[NH], const float (&lv)[NH]) {
#pragma unroll
                for (int h = 0; h < NH; h++)
                    if (h < ng) {
                        if (tg < kv.hd) a.out[(h0 + h) * kv.hd + tg] = lv[h] > 0.f ? ov[h] / lv[h] : 0.f;
                        if (tg == h) {
                            if (a.lse) a.lse[h0 + h] = lv[h] > 0.f ? mv[h] * 0.6931471805599453f + logf(lv[h]) : -INFINITY;
                            if (a.acc_out) {
                                a.ml[2 * (h0 + h)] = mv[h];
                                a.ml[2 * (h0 + h) + 1] = lv[h];
                            }
                        }
                    }
            };
            if (wk.t1 == wk.nt && tg == 0) a.cnt[static_cast<long long>(wk.b) * segs + wk.seg] = cut_of(wk, T, G);
            if (wk.t0 == 0 && wk.t1 == wk.nt) {   // the whole segment
                write_out(o, m, L);
                continue;
            }
            float *part = part_at(a, blockIdx.x, wk.t0 == 0);
#pragma unroll
            for (int h = 0; h < NH; h++) {
                part[h * 128 + tg] = o[h];
                if (tg == h) {
                    part[kAttendPart - 32 + h] = m[h];
                    part[kAttendPart - 16 + h] = L[h];
                }
            }
        }
    }
    __syncthreads();
    if (warp == kWarpO)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
}

template <bool BF, int NH>
cudaError_t launch(const PagedAttendArgs &a, const CUtensorMap &mk, const CUtensorMap &mv, int grid, cudaStream_t st) {
    constexpr int smem = Cfg<BF, NH>::smem;
    static_assert(smem <= 227 * 1024 - 6 * 1024, "shared memory");
    cudaError_t e = allow_smem<k_attend_tc<BF, NH>>(smem);
    if (e != cudaSuccess) return e;
    e = launch_pdl(k_attend_tc<BF, NH>, dim3(grid), dim3(kThreads), smem, st, a, mk, mv);
    return e != cudaSuccess ? e : launch_attend_finish(a, NH, 128, st);
}

}  // namespace

cudaError_t launch_attend_tc(const PagedAttendArgs &a, const CUtensorMap &mk, const CUtensorMap &mv, int sms, cudaStream_t st) {
    const int nh = a.gqa <= 8 ? 8 : 16, grid = attend_grid(a, nh, sms);
    if (a.kv.dtype == STYX_BF16) return nh == 8 ? launch<true, 8>(a, mk, mv, grid, st) : launch<true, 16>(a, mk, mv, grid, st);
    return nh == 8 ? launch<false, 8>(a, mk, mv, grid, st) : launch<false, 16>(a, mk, mv, grid, st);
}

}  // namespace styx
