// Rotary positions as an operator of its own, and the append of keys and values to the paged cache with the rotation
// applied on the way (in the model's own layers the rotation is part of attn_prep_kernel, attention.cu, together with
// the head norms; volundr.py:663-664, batch.py:224-259). Here: half and interleaved layouts, any even part of a head,
// frequencies from a table (so every scaling for long contexts is the table's matter), bf16 or fp16, strided inputs, a
// rotation position apart from the cache slot (a sequence whose first tokens are a prefix held elsewhere).
//
//   angle_i = pos * freq_i;  (u, v) -> m (u cos - v sin, u sin + v cos);  inverse: the transposed rotation.
//
// The angle is a product of a 32-bit integer and a 64-bit frequency: it is formed and reduced to a fraction of a turn in
// double (one rounding of 2^-53 of the turns: 3e-11 turns at a position of 2^18 and frequency 1), then sine and cosine of the
// fraction are taken in fp32. A rotated element is two fp32 products and one rounding to the storage type.
#include "common.cuh"
#include <cuda_fp16.h>

namespace {

// Many small CTAs: a CTA's chain of position, sines and data has little in flight, so as many as the SM holds. 16384 rows of 40
// heads of 128 (336 MB): 512 threads 129 us, 256 94 us, 128 84 us, 128 with the registers held to 32 76 us (4.4 TB/s). Rows
// walked by fewer CTAs, with more loads a thread and 64 to 126 registers, took 121 to 213 us.
constexpr int kRopeThreads = 128, kRopeCtas = 16;
constexpr int kRopeMaxPairs = 512;

template <typename T> __device__ __forceinline__ float to_f(T x);
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float to_f<__half>(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }

template <typename T, int VEC> struct alignas(VEC * 2) Vec { T e[VEC]; };

struct RopeRows {   // [rows, n heads, D]; strides in elements
    const void* src;
    void* dst;      // null: the row goes to a page (below)
    long long src_row, src_head, dst_row, dst_head;
    int n;
    int turn;       // 0: copied as it is
};
struct RopeParams {
    RopeRows s[3];  // q, k, v (rope: the first only)
    void* pool[3];  // null, K, V
    const int* table;
    const int* pos;
    const int* slot;   // null: pos
    const int* seq;    // null: the row's own index
    const double* freq;
    int D, dims, interleaved, inverse, heads, KVH, n_seqs, max_pages, n_pages, paged;
    float magnitude;
};

// One CTA per row (gridDim.y shares of its items). An item is VEC elements of a head together with their partners: in the
// half layout two pieces half a rotation apart, otherwise one piece. Everything is moved once; what bounds the kernel
// is HBM from a few hundred rows on, and the latency of one load -> sine -> store chain below that.
template <typename T, int VEC>
__global__ void __launch_bounds__(kRopeThreads, kRopeCtas) rope_rows_kernel(const RopeParams p) {
    __shared__ float2 cs[kRopeMaxPairs];
    __shared__ int s_page;
    pdl_wait();
    pdl_launch_dependents();
    const long long row = blockIdx.x;
    const int pos = p.pos[row];
    int slot = 0;
    if (p.paged) {
        slot = p.slot ? p.slot[row] : pos;
        if (slot < 0) return;   // a padded row: nothing of it is written
        if (threadIdx.x == 0) {
            const int seq = p.seq ? p.seq[row] : (int)row;
            int page = -1;
            if (seq >= 0 && seq < p.n_seqs && slot / 64 < p.max_pages) page = p.table[(long long)seq * p.max_pages + slot / 64];
            if (page < 0 || page >= p.n_pages) {
                if (blockIdx.y == 0) vk_set_status(VK_ST_BAD_INDEX);
                page = -1;
            }
            s_page = page;
        }
    }
    const int half = p.dims / 2;
    for (int i = threadIdx.x; i < half; i += kRopeThreads) {
        const double turns = (double)pos * p.freq[i] * 0.15915494309189533577;   // 1 / (2 pi)
        const float f = (float)(turns - rint(turns));
        float sn, c;
        sincospif(2.f * f, &sn, &c);
        cs[i] = make_float2(c * p.magnitude, p.inverse ? -sn * p.magnitude : sn * p.magnitude);
    }
    __syncthreads();
    const int page = p.paged ? s_page : 0;
    const int D = p.D;
    const bool pairs = VEC == 1 || !p.interleaved;
    const int step = p.interleaved ? 2 : 1, away = p.interleaved ? 1 : half;   // (interleaved pairs: VEC = 1 only)
    // items of a head: half / VEC pairs of pieces, then the rest of the head; interleaved pieces hold their own partners
    const int npair = pairs ? half / VEC : 0;
    const int per = npair + (D - (pairs ? p.dims : 0)) / VEC;
    const int total = p.heads * per;
    for (int it = blockIdx.y * kRopeThreads + threadIdx.x; it < total; it += kRopeThreads * gridDim.y) {
        int hd = it / per, j = it - hd * per;
        int w = 0;
        while (hd >= p.s[w].n) hd -= p.s[w++].n;
        const RopeRows& s = p.s[w];
        const T* src = (const T*)s.src + row * s.src_row + hd * s.src_head;
        T* dst;
        if (p.pool[w]) {
            if (page < 0) continue;
            dst = (T*)p.pool[w] + (((long long)page * p.KVH + hd) * 64 + (slot & 63)) * D;
        } else {
            dst = (T*)s.dst + row * s.dst_row + hd * s.dst_head;
        }
        if (j < npair) {
            const int i0 = j * VEC, at = i0 * step;
            Vec<T, VEC> a = *reinterpret_cast<const Vec<T, VEC>*>(src + at);
            Vec<T, VEC> b = *reinterpret_cast<const Vec<T, VEC>*>(src + at + away);
            if (s.turn) {
#pragma unroll
                for (int e = 0; e < VEC; e++) {
                    const float2 c = cs[i0 + e];
                    const float u = to_f(a.e[e]), v = to_f(b.e[e]);
                    a.e[e] = from_f<T>(u * c.x - v * c.y);
                    b.e[e] = from_f<T>(u * c.y + v * c.x);
                }
            }
            *reinterpret_cast<Vec<T, VEC>*>(dst + at) = a;
            *reinterpret_cast<Vec<T, VEC>*>(dst + at + away) = b;
        } else {
            const int d0 = (pairs ? p.dims : 0) + (j - npair) * VEC;
            Vec<T, VEC> a = *reinterpret_cast<const Vec<T, VEC>*>(src + d0);
            if constexpr (VEC > 1) {
                if (s.turn && !pairs) {
#pragma unroll
                    for (int e = 0; e < VEC; e += 2) {
                        if (d0 + e < p.dims) {
                            const float2 c = cs[(d0 + e) >> 1];
                            const float u = to_f(a.e[e]), v = to_f(a.e[e + 1]);
                            a.e[e] = from_f<T>(u * c.x - v * c.y);
                            a.e[e + 1] = from_f<T>(u * c.y + v * c.x);
                        }
                    }
                }
            }
            *reinterpret_cast<Vec<T, VEC>*>(dst + d0) = a;
        }
    }
}

template <typename T> cudaError_t rope_launch(int vec, const RopeParams& p, int rows, int ysplit, cudaStream_t stream) {
    const dim3 grid((unsigned)rows, (unsigned)ysplit), block(kRopeThreads);
    if (vec == 8) return vk_launch(rope_rows_kernel<T, 8>, grid, block, 0, stream, p);
    if (vec == 2) return vk_launch(rope_rows_kernel<T, 2>, grid, block, 0, stream, p);
    return vk_launch(rope_rows_kernel<T, 1>, grid, block, 0, stream, p);
}

// The widest piece every pointer and stride allows: 16 bytes, 4 bytes or one element.
// (16384 rows of 40 heads of 128, interleaved: 77 us with 16 bytes, 175 with 4, 173 with one element; the append of 16380 rows in
// the half layout 87, 148, 247)
struct PieceRule {
    uintptr_t bits = 0;
    void rows(const void* p, long long row, long long head) { bits |= (uintptr_t)p | (uintptr_t)(row * 2) | (uintptr_t)(head * 2); }
    int vec(int D, int dims, int interleaved) const {
        const uintptr_t b = bits | (uintptr_t)(D * 2) | (interleaved ? 0 : (uintptr_t)dims);   // half a rotation is dims bytes
        return (b & 15) == 0 ? 8 : (b & 3) == 0 ? 2 : 1;
    }
};

bool rope_shape_ok(int dtype, int rows, int D, int dims, const double* freq, float magnitude) {
    if ((dtype != VK_BF16 && dtype != VK_FP16) || rows < 0 || D <= 0 || D > 1024) return false;
    if (dims < 0 || dims % 2 != 0 || dims > D || (dims > 0 && freq == nullptr)) return false;
    return magnitude == magnitude;
}

// Shares of a row's items over gridDim.y: one pass of the block per share while the grid is small.
int rope_ysplit(int rows, int items) {
    int y = 1;
    while (y < 8 && y * kRopeThreads < items && (long long)rows * y < 148 * 4) y *= 2;
    return y;
}

}  // namespace

extern "C" {

struct vk_rope_args {
    int dtype, rows, heads, D, dims, interleaved, inverse;
    float magnitude;
    const void* x;
    long long x_row, x_head;
    void* out;
    long long out_row, out_head;
    const int* pos;
    const double* freq;
};

struct vk_append_args {
    int dtype, rows, Hq, KVH, D, dims, interleaved;
    float magnitude;
    const void *q, *k, *v;
    long long q_row, q_head, k_row, k_head, v_row, v_head;
    void* q_out;
    long long qo_row, qo_head;
    void *K, *V;
    const int *table, *pos, *slot, *seq;
    const double* freq;
    int n_seqs, max_pages, n_pages;
};

int vk_rope(const vk_rope_args* a, cudaStream_t stream) {
    if (a == nullptr || !rope_shape_ok(a->dtype, a->rows, a->D, a->dims, a->freq, a->magnitude) || a->heads <= 0 || a->heads > 65536) return VK_EINVAL;
    if (a->x_row < 0 || a->x_head < 0 || (a->rows > 1 && a->out_row < a->D) || (a->heads > 1 && a->out_head < a->D)) return VK_EINVAL;
    if (a->rows == 0) return VK_OK;
    if (a->x == nullptr || a->out == nullptr || a->pos == nullptr) return VK_EINVAL;
    if (((uintptr_t)a->x | (uintptr_t)a->out) & 1) return VK_EINVAL;
    RopeParams p = {};
    p.s[0] = RopeRows{a->x, a->out, a->x_row, a->x_head, a->out_row, a->out_head, a->heads, 1};
    p.pos = a->pos; p.freq = a->freq; p.D = a->D; p.dims = a->dims; p.interleaved = a->interleaved != 0; p.inverse = a->inverse != 0;
    p.magnitude = a->magnitude; p.heads = a->heads;
    PieceRule r;
    r.rows(a->x, a->x_row, a->x_head);
    r.rows(a->out, a->out_row, a->out_head);
    const int vec = r.vec(a->D, a->dims, a->interleaved);
    const int ys = rope_ysplit(a->rows, a->heads * ((a->D + vec - 1) / vec));
    return (int)(a->dtype == VK_BF16 ? rope_launch<__nv_bfloat16>(vec, p, a->rows, ys, stream) : rope_launch<__half>(vec, p, a->rows, ys, stream));
}

int vk_kv_append(const vk_append_args* a, cudaStream_t stream) {
    if (a == nullptr || !rope_shape_ok(a->dtype, a->rows, a->D, a->dims, a->freq, a->magnitude)) return VK_EINVAL;
    if (a->KVH <= 0 || a->KVH > 4096 || a->Hq < 0 || a->Hq > 65536 || a->n_seqs <= 0 || a->max_pages <= 0 || a->n_pages <= 0) return VK_EINVAL;
    if (a->k_row < 0 || a->k_head < 0 || a->v_row < 0 || a->v_head < 0) return VK_EINVAL;
    const bool hasq = a->q != nullptr;
    if (hasq != (a->q_out != nullptr) || (hasq && a->Hq == 0)) return VK_EINVAL;
    if (hasq && (a->q_row < 0 || a->q_head < 0 || (a->rows > 1 && a->qo_row < a->D) || (a->Hq > 1 && a->qo_head < a->D))) return VK_EINVAL;
    if (a->seq == nullptr && a->rows > a->n_seqs) return VK_EINVAL;
    if (a->rows == 0) return VK_OK;
    if (!a->k || !a->v || !a->K || !a->V || !a->table || !a->pos) return VK_EINVAL;
    if (((uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)a->K | (uintptr_t)a->V | (uintptr_t)a->q | (uintptr_t)a->q_out) & 1) return VK_EINVAL;
    RopeParams p = {};
    PieceRule r;
    int n = 0;
    if (hasq) {
        p.s[n++] = RopeRows{a->q, a->q_out, a->q_row, a->q_head, a->qo_row, a->qo_head, a->Hq, 1};
        r.rows(a->q, a->q_row, a->q_head);
        r.rows(a->q_out, a->qo_row, a->qo_head);
    }
    p.pool[n] = a->K;
    p.s[n++] = RopeRows{a->k, nullptr, a->k_row, a->k_head, 0, 0, a->KVH, 1};
    p.pool[n] = a->V;
    p.s[n++] = RopeRows{a->v, nullptr, a->v_row, a->v_head, 0, 0, a->KVH, 0};
    r.rows(a->k, a->k_row, a->k_head);
    r.rows(a->v, a->v_row, a->v_head);
    r.rows(a->K, 0, 0);
    r.rows(a->V, 0, 0);
    p.pos = a->pos; p.slot = a->slot; p.seq = a->seq; p.table = a->table; p.freq = a->freq;
    p.D = a->D; p.dims = a->dims; p.interleaved = a->interleaved != 0; p.magnitude = a->magnitude;
    p.heads = (hasq ? a->Hq : 0) + 2 * a->KVH; p.KVH = a->KVH;
    p.n_seqs = a->n_seqs; p.max_pages = a->max_pages; p.n_pages = a->n_pages; p.paged = 1;
    const int vec = r.vec(a->D, a->dims, a->interleaved);
    const int ys = rope_ysplit(a->rows, p.heads * ((a->D + vec - 1) / vec));
    return (int)(a->dtype == VK_BF16 ? rope_launch<__nv_bfloat16>(vec, p, a->rows, ys, stream)
                                     : rope_launch<__half>(vec, p, a->rows, ys, stream));
}

}  // extern "C"
