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

// A unit of work is 128 keys of one kv head against a tile of (row, query head) pairs. Two forms:
//   wide   up to 128 pairs, one tensor-memory lane each: S[128 x 64] = Q K^T (tcgen05.mma, Q and K in shared memory),
//          P = exp2(S - m) in registers, O[128 x D] += P V with P in tensor memory (over S) and V in shared memory. Two
//          streams (a softmax warpgroup and a warp that issues its MMAs each) share the tensor core: two tiles on the same keys,
//          or one tile on the two 64-key halves of every unit;
//   narrow up to 64 pairs (a sequence's own keys, a small batch): mma.sync m16n8k16 by one warpgroup, the unit's keys dealt to
//          its warps in chunks of 32, each warp with its own running maximum, sum and output, joined when the job ends.
//          The two warpgroups take jobs in turn, so that one's start and end lie under the other's units. No round trips
//          between warps and tensor core, and a 16-row tile does not pay for 128.
// A job is a run of units: a tile, or two tiles that share the keys, against the prefix or against one sequence's own keys.
// All jobs lie on one line, each as long as it is expected to take, and every CTA takes an equal interval of it.
constexpr int kPfKeys = 128, kPfNarrow = 64;   // (with the wide form for everything four of the cases took 80 / 120 / 91 / 557 us, with both 54 / 56 / 63 / 196)
// Measured (128 rows x 40 heads of 128 behind 32768 keys, 16 to 1024 own): 137 us, 52 at the tensor core's rate; prefix alone 111,
// own keys alone 43 (131 MB). The prefix takes 2600 cycles per 64 keys of two tiles where its MMAs take 1330 and its softmax
// 1300 a stream: what bounds it is the chain of a stream (scores -> softmax -> P -> next scores), which two S buffers do not
// cover. With S in one buffer of 128 keys a stream the same took 152 us. 16 rows behind 20000 keys: 45 us, 20 at HBM's
// rate; about 13 us of it are the start (lengths, the line, the first job, its queries and keys: one round trip after
// another) and 5 the merge.
// warps 0-3 and 4-7: softmax of two streams; 8: copies; 9, 11: MMAs of the streams; 10: walks the line of work and hands out the
// jobs. The third warpgroup's registers go to the softmax and the narrow form: 168 a thread at launch, then 216 + 216 + 72
constexpr int kPfThreads = 384;
constexpr int kPfSoftmaxRegs = 216, kPfOtherRegs = 72;
// Probabilities meet the values in the storage type. They are at most 2^8 (below); as fp16 they are raised by 2^7, which keeps
// those down to 2^-21 of the largest above fp16's subnormal numbers (bf16 has fp32's range).
template <typename T> constexpr float kPfRaise = std::is_same<T, __half>::value ? 7.f : 0.f;
constexpr int kPfJobs = 4;               // jobs handed out ahead
// Lengths on the line of work: a job's fixed part, a unit of one tile, of two tiles, of the narrow form
struct PfCost { int fixed, one, two; };

template <int D> struct PfCfg {
    static constexpr int kTileBytes = 128 * D * 2;
    static constexpr int kStages = D == 128 ? 5 : 10;
    static constexpr int kSmem = (2 + kStages) * kTileBytes + 1024;
};

struct PfParams {
    CUtensorMap mapK, mapV;
    vk_prefix_args a;
    int G, MT, ST;             // query heads per kv head; tiles of the prefix part, of a sequence's own part
    int narrowP, narrowO;      // the form of either part
    PfCost costP, costO;
    int rowsP, rowsO;          // rows of a slot (a slot holds one job's partial result of one CTA)
    int longest;               // longest unit
    int *head, *cum;           // workspace: {share, longer shares, prefix length}; where a sequence's jobs begin
    float2 *mlP, *mlO;         // running maximum (log2 units) and sum
    float *oP, *oO;            // unnormalised output
};

struct PfJob {
    int kind;                  // -1: no more; bit 0: own pages; bit 1: two tiles; bit 2: narrow
    int h, b, grp, u0, u1, slot, keys;
    __device__ __forceinline__ bool own() const { return kind & 1; }
    __device__ __forceinline__ int tiles() const { return kind & 2 ? 2 : 1; }
    __device__ __forceinline__ bool narrow() const { return kind & 4; }
};

// The line dealt to n CTAs: equal shares, the first `rem` one longer. No share is shorter than the longest unit (n is chosen
// so), hence every CTA between those of a job's first and last unit has a unit of it.
struct PfDeal {
    int q, rem;
    __device__ __forceinline__ int low(int c) const { return c * q + min(c, rem); }
    __device__ __forceinline__ int cta_of(int x) const {
        const int edge = rem * (q + 1);
        return x < edge ? x / (q + 1) : rem + (x - edge) / q;
    }
};

// Units of a job that begin (behind its fixed part) inside [lo, hi), both relative to the job's start
__device__ __forceinline__ void pf_units(int fixed, int w, int nu, int lo, int hi, int& u0, int& u1) {
    u0 = lo <= fixed ? 0 : min(nu, (lo - fixed + w - 1) / w);
    u1 = hi <= fixed ? 0 : min(nu, (hi - fixed + w - 1) / w);
}

// Where the jobs of one kv head lie: tile groups one after another, all of two tiles but perhaps the last
struct PfHead {
    int groups, len2, len, nu;     // tile groups; length of a group of two; of all groups
    __device__ __forceinline__ PfHead(int tiles, int nu_, const PfCost& c) {
        groups = (tiles + 1) / 2;
        nu = nu_;
        len2 = c.fixed + c.two * nu;
        len = nu == 0 ? 0 : (tiles / 2) * len2 + (tiles & 1) * (c.fixed + c.one * nu);
    }
};

__device__ __forceinline__ int pf_clamp(int n, int pages) {
    const int cap = pages * 64;
    if (n > cap) { vk_set_status(VK_ST_BAD_INDEX); n = cap; }
    return n < 0 ? 0 : n;
}

// Keys of sequence b's own pages that any of its rows sees
__device__ __forceinline__ int pf_own_keys(const vk_prefix_args& a, int b) {
    int n = 0;
    for (int t = 0; t < a.T; t += 8) {      // (eight loads at once: one after another a window of eight tokens took 3 us)
        int v[8];
#pragma unroll
        for (int u = 0; u < 8; u++) v[u] = t + u < a.T ? a.lens[b * a.T + t + u] : 0;
#pragma unroll
        for (int u = 0; u < 8; u++) n = max(n, v[u]);
    }
    return pf_clamp(n, a.max_pages);
}
__device__ __forceinline__ int pf_nu(int keys) { return (keys + kPfKeys - 1) / kPfKeys; }

struct PfShared {
    uint64_t full[10], empty[10], qfull[2], sready[2][2], pready[2][2], pvdone[2][2], join[2], njoin[2], nturn[2], jfull[kPfJobs], jempty[kPfJobs];
    PfJob jobs[kPfJobs];
    int lo, hi, cb0, b0, P, fail;
    uint32_t tmem;
    int red[kPfThreads / 32];
    int keys[32];              // of the sequences from b0 on
    float2 ml[8][16];
};

// The jobs of [s.lo, s.hi), one after another: walked by a whole warp, lane i holding the key count of sequence window + i
struct PfIter {
    int cur, hi, cb, b, prefixEnd, window, mine, lane;
    __device__ __forceinline__ void look(const PfParams& p, int from) {
        window = from;
        mine = from + lane < p.a.seqs ? pf_own_keys(p.a, from + lane) : 0;
    }
    __device__ __forceinline__ void init(const PfParams& p, const PfShared& s, int lane_) {
        lane = lane_;
        prefixEnd = PfHead(p.MT, pf_nu(s.P), p.costP).len * p.a.KVH;
        cur = s.lo; hi = s.hi;
        b = s.b0; cb = s.cb0;
        window = b;
        mine = s.keys[lane];
    }
    __device__ __forceinline__ bool next(const PfParams& p, const PfShared& s, PfJob& j) {
        while (cur < hi) {
            int A = 0;
            const bool own = cur >= prefixEnd;
            j.b = 0;
            j.keys = s.P;
            if (own) {
                for (;;) {
                    if (b - window >= 32) look(p, b);
                    j.keys = __shfl_sync(0xffffffffu, mine, b - window);
                    const int len = PfHead(p.ST, pf_nu(j.keys), p.costO).len * p.a.KVH;
                    if (cur < cb + len) break;
                    cb += len;
                    b++;
                }
                j.b = b;
                A = cb;
            }
            const PfCost& c = own ? p.costO : p.costP;
            const int tiles = own ? p.ST : p.MT;
            const PfHead hd(tiles, pf_nu(j.keys), c);
            j.h = (cur - A) / hd.len;
            A += j.h * hd.len;
            j.grp = (cur - A) / hd.len2;
            A += j.grp * hd.len2;
            const bool two = 2 * j.grp + 1 < tiles;
            j.kind = (own ? 1 : 0) | (two ? 2 : 0) | ((own ? p.narrowO : p.narrowP) ? 4 : 0);
            const int w = two ? c.two : c.one, e = min(hi, A + c.fixed + w * hd.nu);
            pf_units(c.fixed, w, hd.nu, cur - A, e - A, j.u0, j.u1);
            j.slot = (j.b * p.a.KVH + j.h) * hd.groups + j.grp + blockIdx.x;
            cur = e;
            if (j.u1 > j.u0) return true;
        }
        j.kind = -1;
        return false;
    }
};

__device__ __forceinline__ void pf_mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// A bounded wait of a whole warp, with one answer for all its lanes
__device__ __forceinline__ bool pf_wait(uint64_t* bar, uint32_t phase) { return __all_sync(0xffffffffu, mbar_wait(bar, phase)); }
// The next job from the queue (a whole warp; lane 0 hands the place back). False at the end or when a wait ran out (then ok too).
__device__ __forceinline__ bool pf_next(PfShared& s, PfJob& j, int& nth, bool& ok) {
    const int q = nth % kPfJobs;
    if (!ok || !pf_wait(&s.jfull[q], (uint32_t)((nth / kPfJobs) & 1))) { ok = false; return false; }
    const int* from = reinterpret_cast<const int*>(&s.jobs[q]);
    int* to = reinterpret_cast<int*>(&j);
#pragma unroll
    for (int i = 0; i < (int)(sizeof(PfJob) / 4); i++) to[i] = __shfl_sync(0xffffffffu, from[i], 0);
    __syncwarp();
    if ((threadIdx.x & 31) == 0) pf_mbar_arrive(&s.jempty[q]);
    nth++;
    return j.kind >= 0;
}
// The calls from here to pf_mma_pv are a whole warp's and one elected lane acts: with warp-uniform operands eight MMAs take 520
// cycles to issue, and 560 to 600 beside the softmax warps of the same scheduler; from inside a branch on the lane,
// 560, and 780 to 950.
#define PF_ELECT ".reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
__device__ __forceinline__ void pf_commit(uint64_t* bar) {
    asm volatile("{\n\t" PF_ELECT "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)) : "memory");
}
// A stage's "empty" barrier counts the four warps of the narrow form; of the wide form's two streams each arrives once now and
// once when its MMAs are done
__device__ __forceinline__ void pf_commit_stage(uint64_t* bar) {
    asm volatile(
        "{\n\t" PF_ELECT "@e mbarrier.arrive.shared::cta.b64 _, [%0];\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar))
        : "memory");
}
// S = Q K^T: descriptors step 32 bytes (16 elements) inside a block of 64 columns, 16 KB to the next
#define PF_QK(off) "add.u64 a, %1, " #off ";\n\tadd.u64 b, %2, " #off ";\n\t@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, t;\n\t"
template <int D> __device__ __forceinline__ void pf_mma_qk(uint32_t d, uint64_t q, uint64_t k, uint32_t idesc) {
    if constexpr (D == 128)
        asm volatile("{\n\t.reg .pred f, t;\n\t.reg .b64 a, b;\n\tsetp.eq.b32 f, %3, 0;\n\tsetp.ne.b32 t, %3, 0;\n\t" PF_ELECT
                     "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, f;\n\t" PF_QK(2) PF_QK(4) PF_QK(6) PF_QK(1024) PF_QK(1026)
                         PF_QK(1028) PF_QK(1030) "}" ::"r"(d), "l"(q), "l"(k), "r"(idesc)
                     : "memory");
    else
        asm volatile("{\n\t.reg .pred f, t;\n\t.reg .b64 a, b;\n\tsetp.eq.b32 f, %3, 0;\n\tsetp.ne.b32 t, %3, 0;\n\t" PF_ELECT
                     "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, f;\n\t" PF_QK(2) PF_QK(4) PF_QK(6) "}" ::"r"(d), "l"(q),
                     "l"(k), "r"(idesc)
                     : "memory");
}
// O (+)= P V over 64 keys: P advances 8 columns of tensor memory, V 16 rows (2 KB) a step
#define PF_PV(pa, vb) "add.u32 a, %1, " #pa ";\n\tadd.u64 b, %2, " #vb ";\n\t@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, t;\n\t"
__device__ __forceinline__ void pf_mma_pv(uint32_t d, uint32_t pm, uint64_t v, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred f, t;\n\t.reg .b64 b;\n\t.reg .b32 a;\n\tsetp.ne.b32 f, %4, 0;\n\tsetp.ne.b32 t, %3, 0;\n\t" PF_ELECT
                 "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, f;\n\t" PF_PV(8, 128) PF_PV(16, 256) PF_PV(24, 384) "}" ::"r"(d),
                 "r"(pm), "l"(v), "r"(idesc), "r"(accumulate)
                 : "memory");
}
__device__ __forceinline__ void pf_ldm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void pf_ldm4t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
template <typename T> __device__ __forceinline__ void pf_mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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
// two fp32 operations an instruction
__device__ __forceinline__ uint64_t pf_two(float lo, float hi) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
    return v;
}
__device__ __forceinline__ void pf_split(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t pf_fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t pf_add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float pf_max_nan(float a, float b) {   // NaN if either is
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
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
__device__ __forceinline__ void pf_ld8(uint32_t addr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];" : PF_R8(r, 0) : "r"(addr));
}
__device__ __forceinline__ void pf_st8(uint32_t addr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::PF_I8(r, 0), "r"(addr) : "memory");
}
__device__ __forceinline__ void pf_ld16(uint32_t addr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : PF_R8(r, 0), PF_R8(r, 8)
                 : "r"(addr));
}
__device__ __forceinline__ void pf_st16(uint32_t addr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::PF_I8(r, 0),
                 PF_I8(r, 8), "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void pf_store8(float* p, const uint32_t* r) {   // 32 bytes: a whole sector per lane
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), PF_I8(r, 0) : "memory");
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

// One step of a stream's softmax (a warp, its lanes' rows of S in tensor memory at tS): 64 scores a row become probabilities,
// in place. nv: scores of the step that the row sees; settled(): waits until the product before has been added to O.
template <typename T, int D, typename Settled>
__device__ __forceinline__ bool pf_softmax(uint32_t tS, uint32_t tO, int nv, bool first, float sl2, float& ref, float& l, Settled settled) {
    constexpr int N = 64;
    // scores the row does not see: -infinity, put into tensor memory eight columns at a time (the last units of a job
    // only; the code of the common path stays small enough for the instruction caches)
    if (__any_sync(0xffffffffu, nv < N)) {
#pragma unroll 1
        for (int c = max(0, __reduce_min_sync(0xffffffffu, nv)) & ~7; c < N; c += 8) {
            uint32_t x[8];
            pf_ld8(tS + c, x);
            pf_wait_ld();
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = c + e < nv ? x[e] : 0xFF800000u;
            pf_st8(tS + c, x);
        }
        pf_wait_st();
    }
    uint32_t r[N];
    float mx[8];
    pf_ld32(tS, r);
    pf_ld32(tS + 32, r + 32);
    pf_wait_ld();
#pragma unroll
    for (int e = 0; e < 8; e++) mx[e] = __uint_as_float(r[e]);
#pragma unroll
    for (int e = 8; e < 32; e++) mx[e & 7] = pf_max_nan(mx[e & 7], __uint_as_float(r[e]));
#pragma unroll
    for (int e = 32; e < 64; e++) mx[e & 7] = pf_max_nan(mx[e & 7], __uint_as_float(r[e]));
#pragma unroll
    for (int e = 4; e > 0; e >>= 1)
#pragma unroll
        for (int k = 0; k < e; k++) mx[k] = pf_max_nan(mx[k], mx[k + e]);
    const float top = mx[0] * sl2;
    // O and l keep their reference until a score exceeds it by 2^8: then both move to the new maximum
    float f = 1.f;
    if (!(top <= ref + 8.f) || ref == -INFINITY) {        // (a NaN score makes the whole row NaN)
        if (ref != -INFINITY) f = pf_ex2(ref - top);
        ref = top;
    }
    if (!first && __any_sync(0xffffffffu, f != 1.f)) {
        if (!settled()) return false;
        l *= f;
#pragma unroll 1
        for (int c = 0; c < D; c += 16) {
            uint32_t o[16];
            pf_ld16(tO + c, o);
            pf_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            pf_st16(tO + c, o);
        }
    }
    const float off = ref == -INFINITY ? 0.f : kPfRaise<T> - ref;
    const uint64_t scale2 = pf_two(sl2, sl2), off2 = pf_two(off, off);
    uint64_t sum2[2] = {0, 0};
#pragma unroll
    for (int c = 0; c < N; c += 2) {
        float e0, e1;
        const uint64_t x = pf_fma2(pf_two(__uint_as_float(r[c]), __uint_as_float(r[c + 1])), scale2, off2);
        pf_split(x, e0, e1);
        e0 = pf_ex2(e0);
        e1 = pf_ex2(e1);
        sum2[(c >> 1) & 1] = pf_add2(sum2[(c >> 1) & 1], pf_two(e0, e1));
        r[c >> 1] = pf_pack<T>(e0, e1);
    }
    pf_st32(tS, r);
    float s0, s1;
    pf_split(pf_add2(sum2[0], sum2[1]), s0, s1);
    l += s0 + s1;
    pf_wait_st();
    return true;
}

// A narrow job, by one warpgroup: 16-row tile warp % wm of the pairs, keys of chunks warp / wm, + 4 / wm, ... of every unit.
// smem: the warpgroup's own 128 D half-words, where the warps' parts meet; turn: narrow jobs before this one; nn: phases of
// s.njoin used so far.
template <typename T, int D>
__device__ __forceinline__ bool pf_narrow(const PfParams& p, PfShared& s, const PfJob& j, uint8_t* smem, const uint8_t* ring, int base, uint32_t turn,
                                          uint32_t& nn) {
    constexpr int NST = PfCfg<D>::kStages, TB = PfCfg<D>::kTileBytes;
    const vk_prefix_args& a = p.a;
    const int sx = threadIdx.x >> 7, warp = (threadIdx.x >> 5) & 3, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const bool own = j.own();
    const int rows = (own ? a.T : a.seqs * a.T) * p.G, keys = j.keys;
    const int wm = rows <= 16 ? 1 : rows <= 32 ? 2 : 4, ng = 4 / wm;
    const int mt = warp % wm, kg = warp / wm;
    const bool work = mt * 16 < rows;
    const float sl2 = a.scale * 1.4426950408889634f;
    // Q as A fragments: rows g and g + 8 of the tile
    uint32_t qa[D / 16][4];
    int see[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int m = mt * 16 + g + 8 * i, r = (own ? j.b * a.T : 0) + m / p.G;
        const bool live = m < rows;
        // (a pair beyond the last: some row's queries, no key seen, nothing written)
        const T* q = (const T*)a.q + (live ? r * a.q_row + (j.h * p.G + m % p.G) * a.q_head : 0);
        see[i] = !live ? 0 : own ? min(keys, max(0, a.lens[r])) : keys;
#pragma unroll
        for (int k = 0; k < D / 16; k++) {
            qa[k][i] = *reinterpret_cast<const uint32_t*>(q + k * 16 + 2 * t);
            qa[k][2 + i] = *reinterpret_cast<const uint32_t*>(q + k * 16 + 8 + 2 * t);
        }
    }
    float o[D / 8][4], ref[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int n = 0; n < D / 8; n++) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
    // A stage's barrier tells only its latest two phases apart, so every warp that waits for a copy must know that the one before
    // it in the same stage has landed: the other warpgroup has seen all of the job before this one.
    bool ok = turn == 0 || pf_wait(&s.nturn[sx ^ 1], ((turn - 1) >> 1) & 1);
    for (int u = j.u0; u < j.u1 && ok; u++) {
        const int ck = base + 2 * (u - j.u0), cv = ck + 1, sk = ck % NST, sv = cv % NST;
        const uint32_t kb = smem_u32(ring + (size_t)sk * TB), vb = smem_u32(ring + (size_t)sv * TB);
        const int kv = min(kPfKeys, keys - u * kPfKeys);
        if (!pf_wait(&s.full[sk], (uint32_t)((ck / NST) & 1)) || !pf_wait(&s.full[sv], (uint32_t)((cv / NST) & 1))) { ok = false; break; }
        if (work) {
#pragma unroll 1
            for (int c = kg; c * 32 < kv; c += ng) {
                float x[4][4] = {};
                const int krow = c * 32 + (lane >> 4) * 8 + (lane & 7);     // K rows as the N side: eight keys a tile
#pragma unroll
                for (int k = 0; k < D / 16; k++) {
                    const int ch = 2 * k + ((lane >> 3) & 1);
                    const uint32_t at = kb + (ch >> 3) * 16384 + krow * 128 + (((ch & 7) ^ (krow & 7)) << 4);
                    uint32_t b[4];
                    pf_ldm4(b, at);
                    pf_mma16<T>(x[0], qa[k], b[0], b[1]);
                    pf_mma16<T>(x[1], qa[k], b[2], b[3]);
                    pf_ldm4(b, at + 16 * 128);
                    pf_mma16<T>(x[2], qa[k], b[0], b[1]);
                    pf_mma16<T>(x[3], qa[k], b[2], b[3]);
                }
                const int key0 = u * kPfKeys + c * 32 + 2 * t;
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    if (__any_sync(0xffffffffu, see[i] < u * kPfKeys + c * 32 + 32)) {
#pragma unroll
                        for (int n = 0; n < 4; n++)
#pragma unroll
                            for (int e = 0; e < 2; e++)
                                if (key0 + 8 * n + e >= see[i]) x[n][2 * i + e] = -INFINITY;
                    }
                    float top = x[0][2 * i];
#pragma unroll
                    for (int n = 0; n < 4; n++) top = fmaxf(top, fmaxf(x[n][2 * i], x[n][2 * i + 1]));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2)) * sl2;
                    float f = 1.f;
                    if (top > ref[i] + 8.f || ref[i] == -INFINITY) {        // (as in the wide form)
                        if (ref[i] != -INFINITY) f = pf_ex2(ref[i] - top);
                        ref[i] = top;
                    }
                    if (__any_sync(0xffffffffu, f != 1.f)) {
                        l[i] *= f;
#pragma unroll
                        for (int n = 0; n < D / 8; n++) { o[n][2 * i] *= f; o[n][2 * i + 1] *= f; }
                    }
                    const float off = ref[i] == -INFINITY ? 0.f : ref[i] - kPfRaise<T>;
#pragma unroll
                    for (int n = 0; n < 4; n++)
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            x[n][2 * i + e] = pf_ex2(fmaf(x[n][2 * i + e], sl2, -off));
                            l[i] += x[n][2 * i + e];
                        }
                }
                if (c * 32 + 32 > kv) {   // values behind the last key may be anything: zeros (0 * NaN is NaN)
                    const int zn = (c * 32 + 32 - kv) * (D / 8);
                    for (int e = lane; e < zn; e += 32) {
                        const int zr = kv + e / (D / 8), ch = e % (D / 8);
                        asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(vb + (ch >> 3) * 16384 + zr * 128 + ((ch & 7) << 4)), "r"(0u) : "memory");
                    }
                    __syncwarp();
                }
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    const uint32_t pa[4] = {pf_pack<T>(x[2 * k][0], x[2 * k][1]), pf_pack<T>(x[2 * k][2], x[2 * k][3]),
                                            pf_pack<T>(x[2 * k + 1][0], x[2 * k + 1][1]), pf_pack<T>(x[2 * k + 1][2], x[2 * k + 1][3])};
                    const int vrow = c * 32 + k * 16 + ((lane >> 3) & 1) * 8 + (lane & 7);   // V rows as the K side, transposed on the way
#pragma unroll
                    for (int n = 0; n < D / 16; n++) {
                        uint32_t b[4];
                        const int ch = 2 * n + (lane >> 4);
                        pf_ldm4t(b, vb + (ch >> 3) * 16384 + vrow * 128 + (((ch & 7) ^ (vrow & 7)) << 4));
                        pf_mma16<T>(o[2 * n], pa, b[0], b[1]);
                        pf_mma16<T>(o[2 * n + 1], pa, b[2], b[3]);
                    }
                }
            }
        }
        __syncwarp();
        if (lane == 0) {
            pf_mbar_arrive(&s.empty[sk]);
            pf_mbar_arrive(&s.empty[sv]);
        }
    }
    if (!ok) return false;
    if (lane == 0) pf_mbar_arrive(&s.nturn[sx]);
    const long long at = (long long)j.slot * (own ? p.rowsO : p.rowsP);
    float2* ml = (own ? p.mlO : p.mlP) + at;
    float* out = (own ? p.oO : p.oP) + at * D;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    }
    if (ng == 1) {                       // every warp has all keys of its rows
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int m = mt * 16 + g + 8 * i;
            if (m < rows) {
                if (t == 0) ml[m] = make_float2(ref[i] - kPfRaise<T>, l[i]);
#pragma unroll
                for (int n = 0; n < D / 8; n++) *reinterpret_cast<float2*>(out + m * D + n * 8 + 2 * t) = make_float2(o[n][2 * i], o[n][2 * i + 1]);
            }
        }
        return true;
    }
    // ---- the warps' parts joined in shared memory, written as the job's partial result
    if (nn > 0 && !pf_wait(&s.njoin[sx], (nn - 1) & 1)) return false;      // the last job's have been read
    float* const buf = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int row = g + 8 * i;
        if (t == 0) s.ml[sx * 4 + warp][row] = make_float2(ref[i] - kPfRaise<T>, l[i]);
#pragma unroll
        for (int n = 0; n < D / 8; n++)   // (blocks of eight columns swapped by row: the eight rows of a store hit different banks)
            *reinterpret_cast<float2*>(buf + (warp * 16 + row) * D + ((n ^ (row & 7)) * 8 + 2 * t)) = make_float2(o[n][2 * i], o[n][2 * i + 1]);
    }
    __syncwarp();
    if (lane == 0) pf_mbar_arrive(&s.njoin[sx]);
    if (!pf_wait(&s.njoin[sx], nn & 1)) return false;
    for (int e = threadIdx.x & 127; e < rows * (D / 4); e += 128) {
        const int m = e / (D / 4), col = (e % (D / 4)) * 4, row = m & 15, w0 = m >> 4;
        float2 x[4];
        float4 v[4];
        float mx = -INFINITY, sum = 0.f;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            if (k < ng) {
                x[k] = s.ml[sx * 4 + w0 + k * wm][row];
                v[k] = *reinterpret_cast<const float4*>(buf + ((w0 + k * wm) * 16 + row) * D + (((col >> 3) ^ (row & 7)) * 8 + (col & 7)));
                mx = fmaxf(mx, x[k].x);
            }
        }
        const float off = mx == -INFINITY ? 0.f : mx;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            if (k < ng) {
                const float f = pf_ex2(x[k].x - off);
                acc.x += v[k].x * f; acc.y += v[k].y * f; acc.z += v[k].z * f; acc.w += v[k].w * f;
                sum += x[k].y * f;
            }
        }
        *reinterpret_cast<float4*>(out + m * D + col) = acc;
        if (col == 0) ml[m] = make_float2(mx, sum);
    }
    __syncwarp();
    if (lane == 0) pf_mbar_arrive(&s.njoin[sx]);
    nn += 2;
    return true;
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
    // (warp index, tensor-memory base and jobs are broadcast, so that the compiler knows them to be the same in all lanes and
    // the MMA warps' operands live in uniform registers)
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;

    if (tid == 0) {
        for (int i = 0; i < NST; i++) { mbar_init(&s.full[i], 1); mbar_init(&s.empty[i], 4); }
        for (int i = 0; i < 2; i++) {
            mbar_init(&s.qfull[i], 128);
            for (int b = 0; b < 2; b++) {
                mbar_init(&s.sready[i][b], 1);
                mbar_init(&s.pready[i][b], 128);
                mbar_init(&s.pvdone[i][b], 1);
            }
            mbar_init(&s.join[i], 8);
            mbar_init(&s.njoin[i], 4);
            mbar_init(&s.nturn[i], 4);
        }
        for (int i = 0; i < kPfJobs; i++) { mbar_init(&s.jfull[i], 1); mbar_init(&s.jempty[i], 11); }
        mbar_fence_init();
        s.fail = 0;
    }
    if (warp == 9) {   // all of tensor memory: S of both streams in columns 0 and 128, O in 256 and 384
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&s.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    pdl_wait();
    pdl_launch_dependents();
    // ---- the line of work: its length, this CTA's interval of it, the sequence in which that starts
    {
        const int chunks = (a.seqs + kPfThreads - 1) / kPfThreads;
        const int P = tid == 0 ? pf_clamp(*a.prefix_len, a.max_prefix_pages) : 0;
        if (tid == 0) s.P = P;
        int keys = 0, before = 0, len = 0;
        // lengths of the sequences' jobs, summed over the block: `before` in front of this thread's sequence, the chunk's sum returned
        auto scan = [&](int c) {
            const int b = c * kPfThreads + tid;
            keys = b < a.seqs ? pf_own_keys(a, b) : 0;
            len = PfHead(p.ST, pf_nu(keys), p.costO).len * a.KVH;
            int v = len;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, v, o);
                if (lane >= o) v += u;
            }
            __syncthreads();
            if (lane == 31) s.red[warp] = v;
            __syncthreads();
            before = v - len;
            int all = 0;
#pragma unroll
            for (int i = 0; i < kPfThreads / 32; i++) {
                if (i < warp) before += s.red[i];
                all += s.red[i];
            }
            return all;
        };
        int all = 0;
        for (int c = 0; c < chunks; c++) all += scan(c);
        const int base = PfHead(p.MT, pf_nu(s.P), p.costP).len * a.KVH, total = base + all;
        const int n = max(1, min((int)gridDim.x, total / p.longest));
        const PfDeal deal = {total / n, total % n};
        const bool has = (int)blockIdx.x < n;
        const int lo = has ? deal.low(blockIdx.x) : total, hi = has ? deal.low(blockIdx.x + 1) : total;
        const int start = max(lo, base);
        if (tid == 0) {
            s.lo = lo;
            s.hi = hi;
            s.b0 = a.seqs;
            s.cb0 = total;
            if (blockIdx.x == 0) { p.head[0] = deal.q; p.head[1] = deal.rem; p.head[2] = P; }
        }
        __syncthreads();
        int running = base;
        for (int c = 0; c < chunks; c++) {
            const int sum = chunks == 1 ? 0 : scan(c);
            const int b = c * kPfThreads + tid, at = running + before;
            if (b < a.seqs) {
                if (blockIdx.x == 0) p.cum[b] = at;
                if (len > 0 && at <= start && start < at + len) { s.b0 = b; s.cb0 = at; }
            }
            running += sum;
        }
        __syncthreads();
        const int i = tid - s.b0;      // (one chunk: the thread of a sequence still has its key count)
        if (chunks == 1) {
            if (i >= 0 && i < 32) s.keys[i] = keys;
        } else if (tid < 32) {
            s.keys[tid] = s.b0 + tid < a.seqs ? pf_own_keys(a, s.b0 + tid) : 0;
        }
    }
    pf_fence_before();
    __syncthreads();
    pf_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, s.tmem, 0);
    PfJob j;
    bool ok = true;
    int nth = 0;

    if (warp >= 8) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPfOtherRegs));
      if (warp == 8) {
        // ---------------------------------------------------------------- copies
        int n = 0;                                   // copies issued so far: stage n % NST
        while (pf_next(s, j, nth, ok)) {
            const int* list = j.own() ? a.table + (long long)j.b * a.max_pages : a.prefix_pages;
            const int pages = (j.keys + 63) / 64, nu = j.u1 - j.u0;
            // page numbers of 32 pages (16 units) at a time, the next 32 already on their way
            int at = j.u0 * 2;
            int ids = at + lane < pages ? list[at + lane] : 0, nxt = at + 32 + lane < pages ? list[at + 32 + lane] : 0;
            int ids0 = at;
            for (int c = 0; c < 2 * nu && ok; c++) {
                const int i = c >> 1, isv = c & 1;
                const int st = n % NST;
                if (n >= NST && !pf_wait(&s.empty[st], (uint32_t)((n / NST - 1) & 1))) { ok = false; break; }
                const int pg = (j.u0 + i) * 2, cnt = min(2, pages - pg);
                if (pg - ids0 >= 32) {
                    ids0 += 32;
                    ids = nxt;
                    nxt = ids0 + 32 + lane < pages ? list[ids0 + 32 + lane] : 0;
                }
                const int rel = pg - ids0;
                const int pid[2] = {__shfl_sync(0xffffffffu, ids, rel), __shfl_sync(0xffffffffu, ids, rel + 1)};
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
      } else if (warp != 10) {
        // ---------------------------------------------------------------- tensor core (the wide form): a warp a stream
        {
            constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
            constexpr uint32_t idesc0 = (1u << 4) | (fmt << 7) | (fmt << 10) | ((128u >> 4) << 24);
            constexpr uint32_t idescO = idesc0 | (1u << 16) | (((uint32_t)D >> 3) << 17);   // V: columns are the N side
            const int sx = warp == 9 ? 0 : 1;
            const uint32_t tS = tmem + sx * 128, tO = tmem + 256 + sx * 128;
            const uint64_t q = pf_desc(smem_u32(smem + sx * TB), 16);
            const uint64_t ring0 = pf_desc(smem_u32(ring), 16);
            constexpr uint64_t kLead = (uint64_t)((16384 - 16) >> 4) << 16;                 // (V: blocks of 64 columns 16 KB apart)
            constexpr uint32_t idescS = idesc0 | ((64u >> 3) << 17);
            int st = 0;                      // the job's first copy: its stage and phase
            uint32_t ph = 0, nq = 0, np[2] = {0, 0};
            auto ahead = [](int& stage, uint32_t& phase, int n) {
                stage += n;
                phase ^= (uint32_t)((stage / NST) & 1);
                stage %= NST;
            };
            while (pf_next(s, j, nth, ok)) {
                const int kind = j.kind, nu = j.u1 - j.u0;
                if (kind & 4) {              // narrow: not for the tensor core
                    ahead(st, ph, 2 * nu);
                    continue;
                }
                // A step is 64 keys: both halves of every unit, one after the other, or this stream's half of it. S has two
                // buffers of 64 columns: the scores of the step after next follow O += P V of this one, so that the softmax
                // never waits for the tensor core's round trip.
                const bool two = kind & 2;
                const int steps = two ? 2 * nu : nu;
                int ks = st, vs = st;        // next K and V copies
                uint32_t kp = ph, vp = ph;
                ahead(vs, vp, 1);
                if (!pf_wait(&s.qfull[sx], nq & 1)) { ok = false; break; }
                nq++;
                for (int k = 0; k < steps + 2; k++) {      // O += P V of step k - 2, then the scores of step k
                    const int b = k & 1, half = two ? b : sx;
                    const bool fresh = !two || b == 0, done = !two || b == 1;   // first, last use of a stage by this stream
                    if (k >= 2) {
                        if ((fresh && !pf_wait(&s.full[vs], vp)) || !pf_wait(&s.pready[sx][b], np[b] & 1)) { ok = false; break; }
                        np[b]++;
                        pf_fence_after();
                        pf_mma_pv(tO, tS + b * 64, ring0 + kLead + (uint64_t)(vs * (TB >> 4) + half * (8192 >> 4)), idescO, k > 2 ? 1u : 0u);
                        if (k >= steps) pf_commit(&s.pvdone[sx][b]);       // (before: the next score product's barrier says so)
                        if (done) {
                            pf_commit_stage(&s.empty[vs]);
                            vs += 2;
                            if (vs >= NST) { vs -= NST; vp ^= 1u; }
                        }
                    }
                    if (k < steps) {
                        if (fresh && !pf_wait(&s.full[ks], kp)) { ok = false; break; }
                        pf_fence_after();
                        pf_mma_qk<D>(tS + b * 64, q, ring0 + (uint64_t)(ks * (TB >> 4) + half * (8192 >> 4)), idescS);
                        pf_commit(&s.sready[sx][b]);
                        if (done) {
                            pf_commit_stage(&s.empty[ks]);
                            ks += 2;
                            if (ks >= NST) { ks -= NST; kp ^= 1u; }
                        }
                    }
                }
                if (!ok) break;
                ahead(st, ph, 2 * nu);
            }
            if (!ok) s.fail = 1;
        }
      } else if (warp == 10) {
        // ---------------------------------------------------------------- jobs
        PfIter it;
        it.init(p, s, lane);
        for (bool more = true; more && ok; nth++) {
            more = it.next(p, s, j);
            const int q = nth % kPfJobs;
            if (nth >= kPfJobs && !pf_wait(&s.jempty[q], (uint32_t)((nth / kPfJobs - 1) & 1))) { ok = false; break; }
            if (lane == 0) {
                s.jobs[q] = j;
                pf_mbar_arrive(&s.jfull[q]);
            }
            __syncwarp();
        }
        if (!ok) s.fail = 1;
      }
    } else {
        // ---------------------------------------------------------------- softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPfSoftmaxRegs));
        const int sx = warp >> 2, row = tid & 127;
        const uint32_t quarter = (uint32_t)(warp & 3) << 21;       // this warp's 32 lanes of tensor memory
        const uint32_t tS = tmem + quarter + sx * 128, tO = tmem + quarter + 256;
        const float sl2 = a.scale * 1.4426950408889634f;
        int base = 0;
        uint32_t ns[2] = {0, 0}, nd[2] = {0, 0}, nj = 0, nn = 0;   // uses of the S buffers, phases of pvdone, joins, phases of njoin
        uint32_t turn = 0;                                         // narrow jobs seen
        while (pf_next(s, j, nth, ok)) {
            const int nu = j.u1 - j.u0, keys = j.keys;
            const bool own = j.own(), two = j.tiles() == 2;
            // what the last jobs left in the streams' Q has been read (pf_narrow looks at its own)
            if (nj > 0 && !pf_wait(&s.join[1], (nj - 1) & 1)) { ok = false; break; }
            if (j.narrow()) {
                if ((int)(turn & 1) == sx) ok = pf_narrow<T, D>(p, s, j, smem + sx * TB, ring, base, turn, nn);
                turn++;
                base += 2 * nu;
                continue;
            }
            if (nn > 0 && !pf_wait(&s.njoin[sx], (nn - 1) & 1)) { ok = false; break; }
            // this thread's (row, query head) pair: lane `row` of the tile
            const int tile0 = (j.grp * 2 + (two ? sx : 0)) * 128, m = tile0 + row;
            const int pairsOf = (own ? a.T : a.seqs * a.T) * p.G;
            const bool live = m < pairsOf;
            int see = 0x7FFFFFFF;                                  // keys it sees (a lane without a pair: zeros, never written)
            const bool work = __any_sync(0xffffffffu, live);
            if (work) {
                const int r = (own ? j.b * a.T : 0) + m / p.G;
                long long qat = -1;
                if (live) {
                    qat = r * a.q_row + (j.h * p.G + m % p.G) * a.q_head;
                    see = own ? min(keys, max(0, a.lens[r])) : keys;
                }
                // the warp's 32 rows of Q, D / 8 lanes a row, into the operand's swizzled layout
                constexpr int LPR = D / 8, RPI = 32 / LPR;
                const int c = lane % LPR;
                uint4 v[32 / RPI];
#pragma unroll
                for (int k = 0; k < 32 / RPI; k++) {
                    const long long at = __shfl_sync(0xffffffffu, qat, k * RPI + lane / LPR);
                    v[k] = reinterpret_cast<const uint4*>((const T*)a.q + (at < 0 ? 0 : at))[c];   // (no branch: all loads in flight at once)
                }
#pragma unroll
                for (int k = 0; k < 32 / RPI; k++) {
                    const int qr = (warp & 3) * 32 + k * RPI + lane / LPR;
                    if (tile0 + qr >= pairsOf) v[k] = make_uint4(0u, 0u, 0u, 0u);
                    *reinterpret_cast<uint4*>(smem + sx * TB + (c >> 3) * 16384 + qr * 128 + (((c & 7) ^ (qr & 7)) << 4)) = v[k];
                }
            }
            fence_proxy_async_smem();
            pf_mbar_arrive(&s.qfull[sx]);

            float ref = -INFINITY, l = 0.f;                        // reference of the exponents (log2 units), sum
            const int steps = two ? 2 * nu : nu;
            for (int i = 0; i < steps; i++) {
                // this step's 64 keys, in a buffer of their own
                const int unit = two ? i >> 1 : i, half = two ? i & 1 : sx, b = i & 1, left = keys - (j.u0 + unit) * kPfKeys - half * 64;
                if (!pf_wait(&s.sready[sx][b], ns[b] & 1)) { ok = false; break; }
                ns[b]++;
                pf_fence_after();
                if (work) {
                    // O += P V of the step before may still be under way when O has to be rescaled. The score product of the
                    // step after this one is issued behind it; the last two steps have a barrier for it.
                    auto settled = [&]() {
                        const bool in = i + 1 < steps ? pf_wait(&s.sready[sx][b ^ 1], ns[b ^ 1] & 1) : pf_wait(&s.pvdone[sx][b ^ 1], nd[b ^ 1] & 1);
                        pf_fence_after();
                        return in;
                    };
                    if (!pf_softmax<T, D>(tS + b * 64, tO + sx * 128, see - keys + left, i == 0, sl2, ref, l, settled)) { ok = false; break; }
                }
                if (left < 64) {
                    // values behind the last key may be anything, and 0 * NaN is NaN: their rows of the stage become zeros
                    // (of two tiles each stream sees to it for itself, whichever comes first)
                    const int c = base + 2 * unit + 1, st = c % NST;
                    if (!pf_wait(&s.full[st], (uint32_t)((c / NST) & 1))) { ok = false; break; }
                    uint8_t* v = ring + (size_t)st * TB + half * 8192;
                    for (int e = max(left, 0) * 8 + row; e < 64 * 8; e += 128)
#pragma unroll
                        for (int x = 0; x < D / 64; x++) *reinterpret_cast<uint4*>(v + x * 16384 + e * 16) = make_uint4(0u, 0u, 0u, 0u);
                    fence_proxy_async_smem();
                }
                pf_fence_before();
                pf_mbar_arrive(&s.pready[sx][b]);
            }
            base += 2 * nu;
            if (!ok) break;
            // ---- the job's partial result
            const int lastb = (steps - 1) & 1;
            if (!pf_wait(&s.pvdone[sx][lastb], nd[lastb] & 1)) { ok = false; break; }
            nd[lastb]++;
            if (steps > 1) nd[lastb ^ 1]++;
            pf_fence_after();
            const int srow = (two ? sx * 128 : 0) + row;
            const long long at = (long long)j.slot * (own ? p.rowsO : p.rowsP) + srow;
            float2* ml = (own ? p.mlO : p.mlP) + at;
            float* o = (own ? p.oO : p.oP) + at * D;
            if (two) {
                if (live) *ml = make_float2(ref - kPfRaise<T>, l);
                if (work) {
#pragma unroll 1
                    for (int c = 0; c < D / 32; c++) {
                        uint32_t r[32];
                        pf_ld32(tO + sx * 128 + c * 32, r);
                        pf_wait_ld();
                        if (live) {
#pragma unroll
                            for (int e = 0; e < 32; e += 8) pf_store8(o + c * 32 + e, r + e);
                        }
                    }
                }
            } else {
                // the two streams' parts of the tile added; each stream's warps write half of the columns
                // (the pairs are exchanged where the streams' Q lay, which no product reads any more)
                reinterpret_cast<float2*>(smem + sx * TB)[row] = make_float2(ref - kPfRaise<T>, l);
                __syncwarp();
                if (lane == 0) pf_mbar_arrive(&s.join[0]);
                if (!pf_wait(&s.join[0], nj & 1)) { ok = false; break; }
                const float2 x0 = reinterpret_cast<const float2*>(smem)[row], x1 = reinterpret_cast<const float2*>(smem + TB)[row];
                const float mx = fmaxf(x0.x, x1.x), off = mx == -INFINITY ? 0.f : mx;
                const float f0 = pf_ex2(x0.x - off), f1 = pf_ex2(x1.x - off);
                if (live && sx == 0) *ml = make_float2(mx, x0.y * f0 + x1.y * f1);
                if (work) {
#pragma unroll 1
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
                            for (int e = 0; e < 32; e += 8) pf_store8(o + col + e, u + e);
                        }
                    }
                }
                pf_fence_before();
                __syncwarp();
                if (lane == 0) pf_mbar_arrive(&s.join[1]);         // (both streams wait for it before they begin another job)
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

// The pieces of one pair's prefix or own part: those of CTAs c0 .. c1 of the line, in the slots' rows at + c * step
struct PfPieces {
    int c0, c1;
    long long at;
};
__device__ __forceinline__ PfPieces pf_pieces(const PfParams& p, bool own, int b, int m, int h, const PfDeal& deal) {
    const vk_prefix_args& a = p.a;
    const int tiles = own ? p.ST : p.MT, grp = m / 256;
    const PfCost& cost = own ? p.costO : p.costP;
    const PfHead hd(tiles, pf_nu(own ? pf_own_keys(a, b) : p.head[2]), cost);
    const int w = 2 * grp + 1 < tiles ? cost.two : cost.one, first = (own ? p.cum[b] : 0) + h * hd.len + grp * hd.len2 + cost.fixed;
    PfPieces x = {0, -1, (long long)((b * a.KVH + h) * hd.groups + grp) * (own ? p.rowsO : p.rowsP) + m - grp * 256};
    if (hd.nu > 0) {
        x.c0 = deal.cta_of(first);
        x.c1 = deal.cta_of(first + w * (hd.nu - 1));
    }
    return x;
}

// out = sum of the pieces of a (row, query head) pair, in the order of the line of work. SPLIT: the eight warps of a CTA share one
// pair's pieces (few pairs: a prefix that all SMs worked on has up to 148 of them); else a warp takes a pair. Both
// are bound by the round trip lengths -> pieces -> sums, four pieces in flight a warp.
template <typename T, int D, bool SPLIT>
__global__ void __launch_bounds__(256) attend_prefix_merge_kernel(const __grid_constant__ PfParams p) {
    constexpr int E = D / 32;
    struct Vec { float v[E]; };
    __shared__ float so[SPLIT ? 8 : 1][D];
    __shared__ float2 sml[8];
    pdl_wait();
    pdl_launch_dependents();
    const vk_prefix_args& a = p.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int pair = SPLIT ? blockIdx.x : blockIdx.x * 8 + warp;
    if (pair >= a.seqs * a.T * a.Hq) return;
    const int r = pair / a.Hq, hq = pair % a.Hq, h = hq / p.G, g = hq % p.G, b = r / a.T;
    if (a.lens[r] < 0) return;
    const PfDeal deal = {p.head[0], p.head[1]};
    float m = -INFINITY, l = 0.f, o[E] = {};
#pragma unroll 1
    for (int own = 0; own < 2; own++) {
        const PfPieces x = own ? pf_pieces(p, true, b, (r - b * a.T) * p.G + g, h, deal) : pf_pieces(p, false, 0, r * p.G + g, h, deal);
        const long long step = own ? p.rowsO : p.rowsP;
        const float2* mls = (own ? p.mlO : p.mlP) + x.at;
        const float* os = (own ? p.oO : p.oP) + x.at * D + lane * E;
        constexpr int STRIDE = SPLIT ? 8 : 1;
        for (int c = x.c0 + (SPLIT ? warp : 0); c <= x.c1; c += 4 * STRIDE) {
            float2 ml[4];
            Vec v[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int cc = c + k * STRIDE;
                ml[k] = make_float2(-INFINITY, 0.f);
                if (cc <= x.c1) {
                    ml[k] = mls[cc * step];
                    if constexpr (E == 4) *reinterpret_cast<float4*>(&v[k]) = *reinterpret_cast<const float4*>(os + cc * step * D);
                    else *reinterpret_cast<float2*>(&v[k]) = *reinterpret_cast<const float2*>(os + cc * step * D);
                } else {
#pragma unroll
                    for (int e = 0; e < E; e++) v[k].v[e] = 0.f;
                }
            }
            const float mn = fmaxf(m, fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x))), off = mn == -INFINITY ? 0.f : mn;
            const float f0 = exp2f(m - off);
            l *= f0;
#pragma unroll
            for (int e = 0; e < E; e++) o[e] *= f0;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const float f = exp2f(ml[k].x - off);
                l += ml[k].y * f;
#pragma unroll
                for (int e = 0; e < E; e++) o[e] += v[k].v[e] * f;
            }
            m = mn;
        }
    }
    if constexpr (SPLIT) {
        if (lane == 0) sml[warp] = make_float2(m, l);
#pragma unroll
        for (int e = 0; e < E; e++) so[warp][lane * E + e] = o[e];
        __syncthreads();
        if (warp != 0) return;
        float mx = -INFINITY;
        for (int i = 0; i < 8; i++) mx = fmaxf(mx, sml[i].x);
        const float off = mx == -INFINITY ? 0.f : mx;
        l = 0.f;
#pragma unroll
        for (int e = 0; e < E; e++) o[e] = 0.f;
        for (int i = 0; i < 8; i++) {
            const float f = exp2f(sml[i].x - off);
            l += sml[i].y * f;
#pragma unroll
            for (int e = 0; e < E; e++) o[e] += so[i][lane * E + e] * f;
        }
    }
    struct alignas(E * 2) Out { T v[E]; } y, gt;
    if (a.gate) gt = *reinterpret_cast<const Out*>((const T*)a.gate + r * a.gate_row + hq * a.gate_head + lane * E);
#pragma unroll
    for (int e = 0; e < E; e++) {
        float v = l == 0.f ? 0.f : o[e] / l;                       // (no visible key: zeros)
        if (a.gate) v /= 1.f + expf(-to_f(gt.v[e]));
        y.v[e] = from_f<T>(v);
    }
    *reinterpret_cast<Out*>((T*)a.out + r * a.out_row + hq * a.out_head + lane * E) = y;
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
    // (eight warps a pair while that gives each SM no more than a few CTAs: 640 pairs of 18 pieces took 13 us longer with a
    // warp each; 5120 pairs of 7 pieces take 13 us with a warp each and 23 with four, caches cold)
    const int pairs = p.a.seqs * p.a.T * p.a.Hq;
    if (pairs <= 8 * sms) return vk_launch(attend_prefix_merge_kernel<T, D, true>, dim3((unsigned)pairs), dim3(256), 0, stream, p);
    return vk_launch(attend_prefix_merge_kernel<T, D, false>, dim3((unsigned)((pairs + 7) / 8)), dim3(256), 0, stream, p);
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
    const long long rows = (long long)a->seqs * a->T;
    if (rows > 65536 || rows * a->Hq > 0x7FFFFFFFll) return VK_ETOOBIG;
    // the line of work (at most 16 a unit of two tiles, as much for a job's fixed part) and the slots are 32-bit counts
    const long long G = a->Hq / a->KVH, gP = (rows * G + 255) / 256, gO = (a->T * G + 255) / 256;
    if (((long long)a->max_prefix_pages / 2 + 2) * a->KVH * gP * 16 + a->seqs * ((long long)a->max_pages / 2 + 2) * a->KVH * gO * 16 > 0x7FFFFFFFll)
        return VK_ETOOBIG;
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
    p.narrowP = mP <= kPfNarrow;
    p.narrowO = mO <= kPfNarrow;
    // (lengths fitted to the times of the CTAs; 1 : 1.2 between the forms, or a fixed part of 6 to 16, changed the cases by 3% and less)
    p.costP = p.costO = PfCost{4, 4, 8};
    p.longest = max(p.MT > 1 ? p.costP.two : p.costP.one, p.ST > 1 ? p.costO.two : p.costO.one);
    p.rowsP = (int)(mP < 256 ? mP : 256);
    p.rowsO = (int)(mO < 256 ? mO : 256);
    const size_t slotsP = (size_t)a->KVH * ((p.MT + 1) / 2) + ctas, slotsO = (size_t)a->seqs * a->KVH * ((p.ST + 1) / 2) + ctas;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        uint8_t* x = ws + at;
        at += (bytes + 255) & ~(size_t)255;
        return x;
    };
    p.head = (int*)take(64);
    p.cum = (int*)take((size_t)a->seqs * 4);
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
