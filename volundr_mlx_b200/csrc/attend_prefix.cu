// Attention of a decode batch whose sequences share a prompt prefix. Row r = b T + t (token t of the T newest of sequence b)
// sees the P keys of the prefix, held once for all sequences in its own list of 64-token pages, and the first lens[r]
// keys of its sequence's pages behind it:  out = softmax(scale q k) v  [times sigmoid(gate)].
#include "common.cuh"
#include <cuda.h>
#include <cuda_fp16.h>
#include <math.h>
#include <type_traits>

extern "C" struct vk_prefix_args {
    int dtype, seqs, T, Hq, KVH, D;
    float scale;
    const void* q;
    long long q_row, q_head;
    const void* gate;
    long long gate_row, gate_head;
    void* out;
    long long out_row, out_head;
    const void *K, *V;
    int n_pages;
    const int* prefix_pages;
    int max_prefix_pages;
    const int* prefix_len;
    const int* table;
    int max_pages;
    const int* lens;
};

namespace {

// A unit of work is 128 keys of one kv head against a tile of up to 128 (row, query head) pairs, one tensor-memory lane each:
//   S[128 x 128] = Q K^T (tcgen05.mma, Q and K in shared memory), P = exp2(S - m) in registers, O[128 x D] += P V with P in
//   tensor memory (over S) and V in shared memory.
// A job is a run of units: a tile, or two tiles that share the keys, against the prefix or against one sequence's own keys.
// All jobs' units lie on one line, weighted by their tiles, and every CTA takes an equal interval of it.
constexpr int kPfTile = 128, kPfKeys = 128;
// warps 0-3 and 4-7: softmax of two streams; 8: copies; 9: tensor core; 10, 11 fill the third warpgroup, whose registers go to
// the softmax (a row of S is 128 registers): 168 a thread at launch, then 216 + 216 + 72 = 3 x 168
constexpr int kPfThreads = 384;
constexpr int kPfSoftmaxRegs = 216, kPfOtherRegs = 72;
constexpr int kPfWindow = 64;            // sequences whose unit counts are kept in shared memory

template <int D> struct PfCfg {
    static constexpr int kTileBytes = 128 * D * 2;
    static constexpr int kStages = D == 128 ? 5 : 10;
    static constexpr int kSmem = (2 + kStages) * kTileBytes + 1024;
};

struct PfParams {
    CUtensorMap mapK, mapV;
    vk_prefix_args a;
    int G, MT, ST;             // query heads per kv head; tiles of the prefix part, of a sequence's own part
    int rowsP, rowsO;          // rows of a slot (a slot holds one job's partial result of one CTA)
    long long *head, *cum;     // workspace: {total, CTAs, prefix length}; exclusive sums of the sequences' unit counts
    float2 *mlP, *mlO;         // running maximum (log2 units) and sum
    float *oP, *oO;            // unnormalised output
};

struct PfJob {
    int own, h, b, grp, u0, u1, tiles;
    long long slot;
};

__device__ __forceinline__ long long pf_low(long long c, long long total, int n) { return c * total / n; }

// The part of a job [A, A + w * units) that lies in [lo, hi): units [u0, u1)
__device__ __forceinline__ void pf_units(long long A, int w, long long lo, long long hi, int& u0, int& u1) {
    u0 = (int)((lo - A + w - 1) / w);
    u1 = (int)((hi - A + w - 1) / w);
}

__device__ __forceinline__ int pf_clamp(int n, int pages) {
    const int cap = pages * 64;
    if (n > cap) { vk_set_status(VK_ST_BAD_INDEX); n = cap; }
    return n < 0 ? 0 : n;
}

// Keys of sequence b's own pages that any of its rows sees
__device__ __forceinline__ int pf_own_keys(const vk_prefix_args& a, int b) {
    int n = 0;
    for (int t = 0; t < a.T; t++) n = max(n, a.lens[(long long)b * a.T + t]);
    return pf_clamp(n, a.max_pages);
}
__device__ __forceinline__ int pf_nu(int keys) { return (keys + kPfKeys - 1) / kPfKeys; }

struct PfShared {
    uint64_t full[10], empty[10], qfull[2], sready[2], pready[2], odone[2], join[2];
    long long total, lo, hi, cb0;
    int b0, P, n, fail;
    uint32_t tmem;
    int keys[kPfWindow];
    long long red[kPfThreads / 32];
};

struct PfIter {
    long long cur, hi, cb;
    int b, keys;
    int npu;
    long long perHead, prefixCost;
    __device__ void init(const PfParams& p, const PfShared& s) {
        npu = pf_nu(s.P);
        perHead = (long long)npu * p.MT;
        prefixCost = perHead * p.a.KVH;
        cur = s.lo; hi = s.hi;
        b = s.b0; cb = s.cb0;
        keys = b < p.a.seqs ? s.keys[0] : 0;
    }
    __device__ int own_keys(const PfParams& p, const PfShared& s, int i) const {
        return i - s.b0 < kPfWindow ? s.keys[i - s.b0] : pf_own_keys(p.a, i);
    }
    __device__ bool next(const PfParams& p, const PfShared& s, PfJob& j) {
        while (cur < hi) {
            long long A, B;
            int w;
            if (cur < prefixCost) {
                j.own = 0; j.b = 0;
                j.h = (int)(cur / perHead);
                j.grp = (int)((cur - j.h * perHead) / (2 * npu));
                w = 2 * j.grp + 1 < p.MT ? 2 : 1;
                A = j.h * perHead + (long long)j.grp * 2 * npu;
                B = A + (long long)w * npu;
                j.slot = (long long)j.h * ((p.MT + 1) / 2) + j.grp;
            } else {
                long long cost;
                int nu;
                for (;;) {
                    nu = pf_nu(keys);
                    cost = (long long)nu * p.a.KVH * p.ST;
                    if (cur < cb + cost) break;
                    cb += cost;
                    b++;
                    keys = own_keys(p, s, b);
                }
                const long long rel = cur - cb, per = (long long)nu * p.ST;
                j.own = 1; j.b = b;
                j.h = (int)(rel / per);
                j.grp = (int)((rel - j.h * per) / (2 * nu));
                w = 2 * j.grp + 1 < p.ST ? 2 : 1;
                A = cb + j.h * per + (long long)j.grp * 2 * nu;
                B = A + (long long)w * nu;
                j.slot = ((long long)b * p.a.KVH + j.h) * ((p.ST + 1) / 2) + j.grp;
            }
            const long long e = hi < B ? hi : B;
            pf_units(A, w, cur, e, j.u0, j.u1);
            j.tiles = w;
            j.slot += blockIdx.x;
            cur = e;
            if (j.u1 > j.u0) return true;
        }
        return false;
    }
};

// Order of a job's copies in the stage ring: as the tensor core uses them (two score products ahead of the values).
__device__ __forceinline__ int pf_stage_k(int i, int tiles) { return tiles == 2 ? 2 * i : (i == 0 ? 0 : 2 * i - 1); }
__device__ __forceinline__ int pf_stage_v(int i, int n, int tiles) { return tiles == 2 ? 2 * i + 1 : (i == n - 1 ? 2 * n - 1 : 2 * i + 2); }

__device__ __forceinline__ void pf_mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// A bounded wait of a whole warp, with one answer for all its lanes
__device__ __forceinline__ bool pf_wait(uint64_t* bar, uint32_t phase) { return __all_sync(0xffffffffu, mbar_wait(bar, phase)); }
__device__ __forceinline__ void pf_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void pf_tma(uint32_t dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
                 "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ float pf_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <typename T> __device__ __forceinline__ uint32_t pf_pack(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pf_pack<__nv_bfloat16>(float lo, float hi) { return pack_bf2(lo, hi); }
template <> __device__ __forceinline__ uint32_t pf_pack<__half>(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

#define PF_R8(r, o) "=r"(r[o]), "=r"(r[o + 1]), "=r"(r[o + 2]), "=r"(r[o + 3]), "=r"(r[o + 4]), "=r"(r[o + 5]), "=r"(r[o + 6]), "=r"(r[o + 7])
#define PF_I8(r, o) "r"(r[o]), "r"(r[o + 1]), "r"(r[o + 2]), "r"(r[o + 3]), "r"(r[o + 4]), "r"(r[o + 5]), "r"(r[o + 6]), "r"(r[o + 7])
// 32 consecutive tensor-memory columns of this thread's lane
__device__ __forceinline__ void pf_ld32(uint32_t addr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, "
        "%19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : PF_R8(r, 0), PF_R8(r, 8), PF_R8(r, 16), PF_R8(r, 24)
        : "r"(addr));
}
__device__ __forceinline__ void pf_st32(uint32_t addr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, "
        "%18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::PF_I8(r, 0),
        PF_I8(r, 8), PF_I8(r, 16), PF_I8(r, 24), "r"(addr)
        : "memory");
}
__device__ __forceinline__ void pf_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void pf_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void pf_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void pf_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Shared-memory operand descriptor: rows of 128 bytes in the 128-byte swizzle, groups of eight rows 1024 bytes apart; `lead`:
// bytes between blocks of 64 columns (used where the columns are the operand's M or N side)
__device__ __forceinline__ uint64_t pf_desc(uint32_t addr, uint32_t lead) {
    return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)(lead >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

template <typename T, int D>
__global__ void __launch_bounds__(kPfThreads, 1) attend_prefix_kernel(const __grid_constant__ PfParams p) {
    using Cfg = PfCfg<D>;
    constexpr int NST = Cfg::kStages, TB = Cfg::kTileBytes;
    extern __shared__ uint8_t pf_smem_raw[];
    __shared__ PfShared s;
    uint8_t* const smem = (uint8_t*)(((uintptr_t)pf_smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* const ring = smem + 2 * TB;
    const vk_prefix_args& a = p.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (tid == 0) {
        for (int i = 0; i < NST; i++) { mbar_init(&s.full[i], 1); mbar_init(&s.empty[i], 1); }
        for (int i = 0; i < 2; i++) {
            mbar_init(&s.qfull[i], 128);
            mbar_init(&s.sready[i], 1);
            mbar_init(&s.pready[i], 128);
            mbar_init(&s.odone[i], 1);
            mbar_init(&s.join[i], 256);
        }
        mbar_fence_init();
        s.fail = 0;
    }
    if (warp == 9) {   // all of tensor memory: S of both streams in columns 0 and 128, O in 256 and 384
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&s.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    pdl_wait();
    pdl_launch_dependents();
    // ---- the line of work: total, this CTA's interval, the sequence in which it starts
    if (tid == 0) s.P = pf_clamp(*a.prefix_len, a.max_prefix_pages);
    const int chunks = (a.seqs + kPfThreads - 1) / kPfThreads;
    long long running = 0;
    for (int pass = 0; pass < 2; pass++) {
        // (pass 0: the total; pass 1: exclusive sums, in which the interval's start is looked up)
        if (pass == 1) {
            if (tid == 0) {
                const long long total = (long long)pf_nu(s.P) * p.MT * a.KVH + running * a.KVH * p.ST;
                s.total = total;
                s.n = (int)(total < gridDim.x ? total : gridDim.x);
                if (s.n > 0 && blockIdx.x < s.n) {
                    s.lo = pf_low(blockIdx.x, total, s.n);
                    s.hi = pf_low(blockIdx.x + 1, total, s.n);
                } else {
                    s.lo = s.hi = total;
                }
                s.b0 = a.seqs;
                s.cb0 = total;
                if (blockIdx.x == 0) { p.head[0] = total; p.head[1] = s.n; p.head[2] = s.P; }
            }
            __syncthreads();
            running = 0;
        }
        for (int c = 0; c < chunks; c++) {
            const int b = c * kPfThreads + tid;
            const int nu = b < a.seqs ? pf_nu(pf_own_keys(a, b)) : 0;
            long long v = nu;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long u = __shfl_up_sync(0xffffffffu, v, o);
                if (lane >= o) v += u;
            }
            if (lane == 31) s.red[warp] = v;
            __syncthreads();
            long long before = running, all = 0;
            for (int i = 0; i < kPfThreads / 32; i++) {
                if (i < warp) before += s.red[i];
                all += s.red[i];
            }
            if (pass == 1 && b < a.seqs) {
                const long long ex = before + v - nu, base = (long long)pf_nu(s.P) * p.MT * a.KVH, per = (long long)a.KVH * p.ST;
                if (blockIdx.x == 0) p.cum[b] = ex;
                // the first sequence with work at or behind the interval's start
                const long long start = s.lo > base ? s.lo : base;
                if (nu > 0 && base + ex * per <= start && start < base + (ex + nu) * per) {
                    s.b0 = b;
                    s.cb0 = base + ex * per;
                }
            }
            running += all;
            __syncthreads();
        }
    }
    if (tid < kPfWindow) s.keys[tid] = s.b0 + tid < a.seqs ? pf_own_keys(a, s.b0 + tid) : 0;
    pf_fence_before();
    __syncthreads();
    pf_fence_after();
    const uint32_t tmem = s.tmem;
    const int P = s.P;
    PfIter it;
    it.init(p, s);
    PfJob j;
    bool ok = true;

    if (warp >= 8) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPfOtherRegs));
      if (warp == 8) {
        // ---------------------------------------------------------------- copies
        int n = 0;                                   // copies issued so far: stage n % NST
        while (ok && it.next(p, s, j)) {
            const int keys = j.own ? it.keys : P;
            const int* list = j.own ? a.table + (long long)j.b * a.max_pages : a.prefix_pages;
            const int pages = (keys + 63) / 64, nu = j.u1 - j.u0;
            // page numbers of 32 pages (16 units) at a time, the next 32 already on their way
            int at = j.u0 * 2;
            int ids = at + lane < pages ? list[at + lane] : 0, nxt = at + 32 + lane < pages ? list[at + 32 + lane] : 0;
            int ids0 = at;
            // copies in the tensor core's order: copy c of the job is K or V of some unit
            for (int c = 0; c < 2 * nu && ok; c++) {
                int i, isv;
                if (j.tiles == 2) { i = c >> 1; isv = c & 1; }
                else if (c == 0) { i = 0; isv = 0; }
                else if (c == 2 * nu - 1) { i = nu - 1; isv = 1; }
                else if (c & 1) { i = (c + 1) >> 1; isv = 0; }
                else { i = (c - 2) >> 1; isv = 1; }
                const int st = n % NST;
                if (n >= NST && !pf_wait(&s.empty[st], (uint32_t)((n / NST - 1) & 1))) { ok = false; break; }
                const int pg = (j.u0 + i) * 2, cnt = min(2, pages - pg);
                // (V trails K by one unit: the window moves on only when V's pages are behind it, so look both up here)
                if (pg - ids0 >= 34) {
                    ids0 += 32;
                    ids = nxt;
                    nxt = ids0 + 32 + lane < pages ? list[ids0 + 32 + lane] : 0;
                }
                const int rel = pg - ids0;
                int pid[2];
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    const int x = __shfl_sync(0xffffffffu, ids, (rel + k) & 31), y = __shfl_sync(0xffffffffu, nxt, (rel + k) & 31);
                    pid[k] = rel + k < 32 ? x : y;
                }
                if (lane == 0) {
                    fence_proxy_async_smem();   // (rows behind the last key are zeroed in the generic proxy)
                    mbar_expect_tx(&s.full[st], (uint32_t)(cnt * 64 * D * 2));
                    for (int k = 0; k < cnt; k++) {
                        int page = pid[k];
                        if (page < 0 || page >= a.n_pages) { vk_set_status(VK_ST_BAD_INDEX); page = 0; }
                        const int y = (page * a.KVH + j.h) * 64;
#pragma unroll
                        for (int x = 0; x < D / 64; x++)
                            pf_tma(smem_u32(ring + (size_t)st * TB + x * 16384 + k * 8192), isv ? &p.mapV : &p.mapK, x * 64, y, &s.full[st]);
                    }
                }
                __syncwarp();
                n++;
            }
        }
        if (!ok) {   // let the copies in flight land
            s.fail = 1;
            for (int k = n > NST ? n - NST : 0; k < n; k++) mbar_wait(&s.full[k % NST], (uint32_t)((k / NST) & 1));
        }
      } else if (warp == 9 && lane == 0) {
        // ---------------------------------------------------------------- tensor core
        {
            constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
            constexpr uint32_t idesc0 = (1u << 4) | (fmt << 7) | (fmt << 10) | ((128u >> 4) << 24);
            constexpr uint32_t idescS = idesc0 | ((128u >> 3) << 17);
            constexpr uint32_t idescO = idesc0 | (1u << 16) | (((uint32_t)D >> 3) << 17);   // V: columns are the N side
            int base = 0;                    // copies of the jobs before this one
            uint32_t nq[2] = {0, 0}, np[2] = {0, 0};
            while (ok && it.next(p, s, j)) {
                const int nu = j.u1 - j.u0, steps = nu * j.tiles;
                auto score = [&](int i) {    // S of stream i & 1 = Q K^T of step i
                    const int sx = i & 1, c = base + pf_stage_k(j.tiles == 2 ? i >> 1 : i, j.tiles), st = c % NST;
                    if (!mbar_wait(&s.full[st], (uint32_t)((c / NST) & 1))) { ok = false; return; }
                    pf_fence_after();
                    const uint32_t q0 = smem_u32(smem + sx * TB), k0 = smem_u32(ring + (size_t)st * TB);
#pragma unroll
                    for (int kk = 0; kk < D / 16; kk++) {
                        const uint32_t off = (kk >> 2) * 16384 + (kk & 3) * 32;
                        const uint64_t da = pf_desc(q0 + off, 16), db = pf_desc(k0 + off, 16);
                        asm volatile(
                            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                            "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(tmem + sx * 128),
                            "l"(da), "l"(db), "r"(idescS), "r"(kk > 0 ? 1u : 0u)
                            : "memory");
                    }
                    if (j.tiles == 1 || sx == 1) pf_commit(&s.empty[st]);
                    pf_commit(&s.sready[sx]);
                };
                for (int x = 0; x < 2 && x < steps && ok; x++) {
                    if (!mbar_wait(&s.qfull[x], nq[x] & 1)) { ok = false; break; }
                    nq[x]++;
                }
                if (ok) score(0);
                if (ok && steps > 1) score(1);
                for (int i = 0; i < steps && ok; i++) {
                    const int sx = i & 1, unit = j.tiles == 2 ? i >> 1 : i;
                    const int c = base + pf_stage_v(unit, nu, j.tiles), st = c % NST;
                    if (!mbar_wait(&s.full[st], (uint32_t)((c / NST) & 1)) || !mbar_wait(&s.pready[sx], np[sx] & 1)) { ok = false; break; }
                    np[sx]++;
                    pf_fence_after();
                    const uint32_t v0 = smem_u32(ring + (size_t)st * TB);
#pragma unroll
                    for (int kk = 0; kk < kPfKeys / 16; kk++) {
                        const uint64_t db = pf_desc(v0 + kk * 2048, 16384);
                        asm volatile(
                            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                            "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(tmem + 256 + sx * 128),
                            "r"(tmem + sx * 128 + kk * 8), "l"(db), "r"(idescO), "r"(i >= 2 || kk > 0 ? 1u : 0u)
                            : "memory");
                    }
                    if (j.tiles == 1 || sx == 1) pf_commit(&s.empty[st]);
                    if (i + 2 >= steps) pf_commit(&s.odone[sx]);
                    else score(i + 2);
                }
                base += 2 * nu;
            }
            if (!ok) s.fail = 1;
        }
      }
    } else {
        // ---------------------------------------------------------------- softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPfSoftmaxRegs));
        const int sx = warp >> 2, row = tid & 127;
        const uint32_t quarter = (uint32_t)(warp & 3) << 21;       // this warp's 32 lanes of tensor memory
        const uint32_t tS = tmem + quarter + sx * 128, tO = tmem + quarter + 256;
        const float sl2 = a.scale * 1.4426950408889634f;
        int base = 0;
        uint32_t ns = 0, no = 0, nj = 0;
        while (ok && it.next(p, s, j)) {
            const int nu = j.u1 - j.u0, steps = nu * j.tiles;
            const int keys = j.own ? it.keys : P;
            const int mine = (steps + 1 - sx) / 2;                 // steps of this stream
            if (mine == 0) { base += 2 * nu; continue; }           // (one unit of one tile: the other stream alone)
            // this thread's (row, query head) pair
            const int tile = j.grp * 2 + (j.tiles == 2 ? sx : 0);
            const long long m = (long long)tile * 128 + row;
            const bool live = m < (long long)(j.own ? a.T : a.seqs * a.T) * p.G;
            int see = 0x7FFFFFFF;                                  // keys it sees (a lane without a pair: zeros, never written)
            uint8_t* const qdst = smem + sx * TB + row * 128;
            const bool work = __any_sync(0xffffffffu, live);
            if (live) {
                const long long r = (j.own ? (long long)j.b * a.T : 0) + m / p.G;
                const T* q = (const T*)a.q + r * a.q_row + (j.h * p.G + m % p.G) * a.q_head;
#pragma unroll
                for (int c = 0; c < D / 8; c++)
                    *reinterpret_cast<uint4*>(qdst + (c >> 3) * 16384 + (((c & 7) ^ (row & 7)) << 4)) = reinterpret_cast<const uint4*>(q)[c];
                see = j.own ? min(keys, max(0, a.lens[r])) : P;
            } else if (work) {
#pragma unroll
                for (int c = 0; c < D / 8; c++)
                    *reinterpret_cast<uint4*>(qdst + (c >> 3) * 16384 + (((c & 7) ^ (row & 7)) << 4)) = make_uint4(0u, 0u, 0u, 0u);
            }
            fence_proxy_async_smem();
            pf_mbar_arrive(&s.qfull[sx]);

            float ref = -INFINITY, l = 0.f;                        // reference of the exponents (log2 units), sum
            for (int i = 0; i < mine && ok; i++) {
                const int unit = j.tiles == 2 ? i : 2 * i + sx, key0 = (j.u0 + unit) * kPfKeys;
                if (!pf_wait(&s.sready[sx], ns & 1)) { ok = false; break; }
                ns++;
                pf_fence_after();
                if (work) {
                    uint32_t r[128];
#pragma unroll
                    for (int c = 0; c < 4; c++) pf_ld32(tS + c * 32, r + c * 32);
                    pf_wait_ld();
                    float x[128];
#pragma unroll
                    for (int c = 0; c < 128; c++) x[c] = __uint_as_float(r[c]);
                    const int nv = see - key0;
                    if (__any_sync(0xffffffffu, nv < kPfKeys)) {
#pragma unroll
                        for (int c = 0; c < 128; c++) x[c] = c < nv ? x[c] : -INFINITY;
                    }
                    float mx[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
                    for (int c = 4; c < 128; c++) mx[c & 3] = fmaxf(mx[c & 3], x[c]);
                    const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * sl2;
                    // O and l keep their reference until a score exceeds it by 2^8: then both move to the new maximum
                    float f = 1.f;
                    if (top > ref + 8.f || ref == -INFINITY) {
                        if (ref != -INFINITY) f = pf_ex2(ref - top);
                        ref = top;
                    }
                    if (i > 0 && __any_sync(0xffffffffu, f != 1.f)) {
                        l *= f;
#pragma unroll
                        for (int c = 0; c < D / 32; c++) {
                            uint32_t o[32];
                            pf_ld32(tO + sx * 128 + c * 32, o);
                            pf_wait_ld();
#pragma unroll
                            for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                            pf_st32(tO + sx * 128 + c * 32, o);
                        }
                    }
                    const float off = ref == -INFINITY ? 0.f : ref;
                    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int c = 0; c < 128; c += 2) {
                        const float e0 = pf_ex2(fmaf(x[c], sl2, -off)), e1 = pf_ex2(fmaf(x[c + 1], sl2, -off));
                        sum[c & 2] += e0;
                        sum[(c & 2) + 1] += e1;
                        r[c >> 1] = pf_pack<T>(e0, e1);
                    }
                    l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                    pf_st32(tS, r);
                    pf_st32(tS + 32, r + 32);
                    pf_wait_st();
                }
                // values behind the last key may be anything, and 0 * NaN is NaN: their rows of the stage become zeros
                const int kv = keys - key0;
                if (kv < kPfKeys && (j.tiles == 1 || sx == 0)) {
                    const int c = base + pf_stage_v(unit, nu, j.tiles), st = c % NST;
                    if (!pf_wait(&s.full[st], (uint32_t)((c / NST) & 1))) { ok = false; break; }
                    uint8_t* v = ring + (size_t)st * TB;
                    for (int e = kv * 8 + row; e < kPfKeys * 8; e += 128)
#pragma unroll
                        for (int x = 0; x < D / 64; x++) *reinterpret_cast<uint4*>(v + x * 16384 + e * 16) = make_uint4(0u, 0u, 0u, 0u);
                    fence_proxy_async_smem();
                }
                pf_fence_before();
                pf_mbar_arrive(&s.pready[sx]);
            }
            base += 2 * nu;
            if (!ok) break;
            // ---- the job's partial result
            if (!pf_wait(&s.odone[sx], no & 1)) { ok = false; break; }
            no++;
            pf_fence_after();
            const bool join = j.tiles == 1 && steps > 1;           // both streams hold a part of the same tile
            const int srow = (j.tiles == 2 ? sx * 128 : 0) + row;
            const long long at = j.slot * (j.own ? p.rowsO : p.rowsP) + srow;
            float2* ml = (j.own ? p.mlO : p.mlP) + at;
            float* o = (j.own ? p.oO : p.oP) + at * D;
            if (!join) {
                if (live) *ml = make_float2(ref, l);
                if (work) {
#pragma unroll
                    for (int c = 0; c < D / 32; c++) {
                        uint32_t r[32];
                        pf_ld32(tO + sx * 128 + c * 32, r);
                        pf_wait_ld();
                        if (live) {
#pragma unroll
                            for (int e = 0; e < 8; e++) reinterpret_cast<uint4*>(o)[c * 8 + e] = make_uint4(r[4 * e], r[4 * e + 1], r[4 * e + 2], r[4 * e + 3]);
                        }
                    }
                }
            } else {
                // the two streams' parts added; each stream's warps write half of the columns
                // (the pairs are exchanged where the streams' Q lay, which no product reads any more)
                reinterpret_cast<float2*>(smem + sx * TB)[row] = make_float2(ref, l);
                pf_mbar_arrive(&s.join[0]);
                if (!pf_wait(&s.join[0], nj & 1)) { ok = false; break; }
                const float2 x0 = reinterpret_cast<const float2*>(smem)[row], x1 = reinterpret_cast<const float2*>(smem + TB)[row];
                const float mx = fmaxf(x0.x, x1.x), off = mx == -INFINITY ? 0.f : mx;
                const float f0 = pf_ex2(x0.x - off), f1 = pf_ex2(x1.x - off);
                if (live && sx == 0) *ml = make_float2(mx, x0.y * f0 + x1.y * f1);
                if (work) {
#pragma unroll
                    for (int c = 0; c < D / 64; c++) {
                        const int col = sx * (D / 2) + c * 32;
                        uint32_t u[32], v[32];
                        pf_ld32(tO + col, u);
                        pf_ld32(tO + 128 + col, v);
                        pf_wait_ld();
                        if (live) {
#pragma unroll
                            for (int e = 0; e < 32; e++) u[e] = __float_as_uint(__uint_as_float(u[e]) * f0 + __uint_as_float(v[e]) * f1);
#pragma unroll
                            for (int e = 0; e < 8; e++) reinterpret_cast<uint4*>(o + col)[e] = make_uint4(u[4 * e], u[4 * e + 1], u[4 * e + 2], u[4 * e + 3]);
                        }
                    }
                }
                pf_fence_before();
                pf_mbar_arrive(&s.join[1]);
                if (!pf_wait(&s.join[1], nj & 1)) { ok = false; break; }   // O and the exchanged pairs are free again
                pf_fence_after();
                nj++;
            }
        }
        if (!ok) s.fail = 1;
    }
    pf_fence_before();
    __syncthreads();
    if (warp == 9) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    if (tid == 0 && s.fail) vk_set_status(VK_ST_MBAR_TIMEOUT);
}

// out = sum of the pieces of a (row, query head) pair, in the order of the line of work: one CTA per pair, four warps share
// the pieces.
template <typename T, int D>
__global__ void __launch_bounds__(128) attend_prefix_merge_kernel(const __grid_constant__ PfParams p) {
    constexpr int E = D / 32;
    __shared__ float so[4][D];
    __shared__ float2 sml[4];
    pdl_wait();
    pdl_launch_dependents();
    const vk_prefix_args& a = p.a;
    const int r = blockIdx.x / a.Hq, hq = blockIdx.x % a.Hq, h = hq / p.G, g = hq % p.G;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (a.lens[r] < 0) return;
    const long long total = p.head[0];
    const int n = (int)p.head[1], npu = pf_nu((int)p.head[2]);
    float m = -INFINITY, l = 0.f, o[E] = {};
    for (int own = 0; own < 2; own++) {
        long long A, slot;
        int w, nu, srow;
        if (own) {
            const int b = r / a.T, mm = (r - b * a.T) * p.G + g, tile = mm / 128, grp = tile / 2;
            nu = pf_nu(pf_own_keys(a, b));
            w = 2 * grp + 1 < p.ST ? 2 : 1;
            A = (long long)npu * p.MT * a.KVH + (p.cum[b] * a.KVH + (long long)h * nu) * p.ST + (long long)grp * 2 * nu;
            slot = ((long long)b * a.KVH + h) * ((p.ST + 1) / 2) + grp;
            srow = mm - grp * 256;
        } else {
            const long long mm = (long long)r * p.G + g, tile = mm / 128, grp = tile / 2;
            nu = npu;
            w = 2 * grp + 1 < p.MT ? 2 : 1;
            A = ((long long)h * p.MT + grp * 2) * npu;
            slot = (long long)h * ((p.MT + 1) / 2) + grp;
            srow = (int)(mm - grp * 256);
        }
        if (nu == 0) continue;
        const long long B = A + (long long)w * nu;
        const int c0 = (int)(((A + 1) * n - 1) / total), c1 = (int)((B * n - 1) / total);
        for (int c = c0 + warp; c <= c1; c += 4) {
            const long long lo = pf_low(c, total, n), hi = pf_low(c + 1, total, n);
            int u0, u1;
            pf_units(A, w, lo > A ? lo : A, hi < B ? hi : B, u0, u1);
            if (u1 <= u0) continue;
            const long long at = (slot + c) * (own ? p.rowsO : p.rowsP) + srow;
            const float2 x = (own ? p.mlO : p.mlP)[at];
            const float* src = (own ? p.oO : p.oP) + at * D;
            const float mn = fmaxf(m, x.x), off = mn == -INFINITY ? 0.f : mn;
            const float f0 = exp2f(m - off), f1 = exp2f(x.x - off);
            l = l * f0 + x.y * f1;
#pragma unroll
            for (int e = 0; e < E; e++) o[e] = o[e] * f0 + src[e * 32 + lane] * f1;
            m = mn;
        }
    }
    if (lane == 0) sml[warp] = make_float2(m, l);
#pragma unroll
    for (int e = 0; e < E; e++) so[warp][e * 32 + lane] = o[e];
    __syncthreads();
    const int d = threadIdx.x;
    if (d >= D) return;
    float mx = -INFINITY, sum = 0.f, v = 0.f;
    for (int i = 0; i < 4; i++) mx = fmaxf(mx, sml[i].x);
    const float off = mx == -INFINITY ? 0.f : mx;
    for (int i = 0; i < 4; i++) {
        const float f = exp2f(sml[i].x - off);
        sum += sml[i].y * f;
        v += so[i][d] * f;
    }
    v = sum == 0.f ? 0.f : v / sum;                                // (no visible key: zeros)
    if (a.gate) v /= 1.f + expf(-to_f(((const T*)a.gate)[r * a.gate_row + hq * a.gate_head + d]));
    ((T*)a.out)[r * a.out_row + hq * a.out_head + d] = from_f<T>(v);
}

typedef CUresult (*PfEncode)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                             const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// Pages as a matrix of key rows; a copy takes 64 rows x 64 columns into the 128-byte swizzle.
cudaError_t pf_map(CUtensorMap* map, const vk_prefix_args* a, const void* pool) {
    static std::atomic<void*> entry{nullptr};
    void* f = entry.load(std::memory_order_acquire);
    if (f == nullptr) {
        cudaDriverEntryPointQueryResult found;
        const cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found);
        if (e != cudaSuccess) return e;
        if (found != cudaDriverEntryPointSuccess || f == nullptr) return cudaErrorNotSupported;
        entry.store(f, std::memory_order_release);
    }
    const cuuint64_t dims[2] = {(cuuint64_t)a->D, (cuuint64_t)a->n_pages * a->KVH * 64}, strides[1] = {(cuuint64_t)a->D * 2};
    const cuuint32_t box[2] = {64, 64}, step[2] = {1, 1};
    const CUresult r = ((PfEncode)f)(map, a->dtype == VK_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
                                     const_cast<void*>(pool), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                     CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

template <typename T, int D> cudaError_t pf_launch(const PfParams& p, int sms, cudaStream_t stream) {
    static PerDeviceOnce once;
    cudaError_t e = once.run([] { return cudaFuncSetAttribute(attend_prefix_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, PfCfg<D>::kSmem); });
    if (e != cudaSuccess) return e;
    e = vk_launch(attend_prefix_kernel<T, D>, dim3((unsigned)sms), dim3(kPfThreads), PfCfg<D>::kSmem, stream, p);
    if (e != cudaSuccess) return e;
    return vk_launch(attend_prefix_merge_kernel<T, D>, dim3((unsigned)(p.a.seqs * p.a.T * p.a.Hq)), dim3(128), 0, stream, p);
}

int prefix_args_ok(const vk_prefix_args* a) {
    if (a == nullptr || (a->dtype != VK_BF16 && a->dtype != VK_FP16) || (a->D != 64 && a->D != 128)) return VK_EINVAL;
    if (a->seqs < 0 || a->T <= 0 || a->KVH <= 0 || a->Hq <= 0 || a->Hq % a->KVH != 0 || !(a->scale > 0.f && a->scale < INFINITY) || a->n_pages <= 0) return VK_EINVAL;
    if (a->max_prefix_pages < 0 || a->max_pages < 0 || !a->prefix_len || !a->lens || !a->K || !a->V || !a->q || !a->out) return VK_EINVAL;
    if ((a->max_prefix_pages > 0 && !a->prefix_pages) || (a->max_pages > 0 && !a->table)) return VK_EINVAL;
    if (a->q_row < 0 || a->q_head < 0 || a->out_row < a->D || a->out_head < a->D) return VK_EINVAL;
    if (((uintptr_t)a->q | (uintptr_t)a->out | (uintptr_t)a->K | (uintptr_t)a->V | (uintptr_t)a->gate) & 15) return VK_EINVAL;
    if ((a->q_row | a->q_head | a->out_row | a->out_head) % 8 != 0) return VK_EINVAL;
    if (a->gate && (a->gate_row < 0 || a->gate_head < 0 || (a->gate_row | a->gate_head) % 8 != 0)) return VK_EINVAL;
    // key rows are addressed by 32-bit coordinates, rows and key counts are 32-bit counts
    if ((long long)a->n_pages * a->KVH * 64 > 0x7FFFFFFFll || (long long)a->max_prefix_pages * 64 > 0x7FFFFFFFll ||
        (long long)a->max_pages * 64 > 0x7FFFFFFFll)
        return VK_ETOOBIG;
    if ((long long)a->seqs * a->T > 65536) return VK_ETOOBIG;
    return VK_OK;
}

// One CTA per SM (148, the target's count, where no device answers).
int pf_ctas() {
    static std::atomic<int> sms{0};
    int n = sms.load(std::memory_order_acquire);
    if (n == 0) {
        int dev = 0;
        if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) {
            cudaGetLastError();
            return 148;
        }
        sms.store(n, std::memory_order_release);
    }
    return n;
}

// Fills the layout of the call's workspace; returns its size. A job's piece of CTA c has the slot (job + c): along the line of
// work each step raises the one or the other, so slots are distinct, and there are jobs + CTAs of them.
size_t pf_layout(PfParams& p, const vk_prefix_args* a, uint8_t* ws, int ctas) {
    p.a = *a;
    p.G = a->Hq / a->KVH;
    const long long mP = (long long)a->seqs * a->T * p.G, mO = (long long)a->T * p.G;
    p.MT = (int)((mP + 127) / 128);
    p.ST = (int)((mO + 127) / 128);
    p.rowsP = (int)(mP < 256 ? mP : 256);
    p.rowsO = (int)(mO < 256 ? mO : 256);
    const size_t slotsP = (size_t)a->KVH * ((p.MT + 1) / 2) + ctas, slotsO = (size_t)a->seqs * a->KVH * ((p.ST + 1) / 2) + ctas;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        uint8_t* x = ws + at;
        at += (bytes + 255) & ~(size_t)255;
        return x;
    };
    p.head = (long long*)take(64);
    p.cum = (long long*)take((size_t)a->seqs * 8);
    p.mlP = (float2*)take(slotsP * p.rowsP * 8);
    p.mlO = (float2*)take(slotsO * p.rowsO * 8);
    p.oP = (float*)take(slotsP * p.rowsP * a->D * 4);
    p.oO = (float*)take(slotsO * p.rowsO * a->D * 4);
    return at;
}

}  // namespace

extern "C" {

size_t vk_attend_prefix_workspace_bytes(const vk_prefix_args* a) {
    PfParams p;
    return prefix_args_ok(a) == VK_OK ? pf_layout(p, a, nullptr, pf_ctas()) : 0;
}

int vk_attend_prefix(const vk_prefix_args* a, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
    const int ok = prefix_args_ok(a);
    if (ok != VK_OK || a->seqs == 0) return ok;
    if (workspace == nullptr || ((uintptr_t)workspace & 15)) return VK_EINVAL;
    PfParams p;
    const int ctas = pf_ctas();
    if (workspace_bytes < pf_layout(p, a, (uint8_t*)workspace, ctas)) return VK_ENOSPC;
    VK_CUDA(pf_map(&p.mapK, a, a->K));
    VK_CUDA(pf_map(&p.mapV, a, a->V));
    if (a->dtype == VK_BF16)
        return (int)(a->D == 128 ? pf_launch<__nv_bfloat16, 128>(p, ctas, stream) : pf_launch<__nv_bfloat16, 64>(p, ctas, stream));
    return (int)(a->D == 128 ? pf_launch<__half, 128>(p, ctas, stream) : pf_launch<__half, 64>(p, ctas, stream));
}

}  // extern "C"
