// Attention of a decode batch whose sequences share a prompt prefix. Row r = b T + t (token t of the T newest of sequence b)
// sees the P keys of the prefix, held once for all sequences in its own list of 64-token pages, and the first lens[r]
// keys of its sequence's pages behind it:  out = softmax(scale q k) v  [times sigmoid(gate)].
#include "common.cuh"
#include <cuda_fp16.h>
#include <math.h>

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

// One warp per (row, query head), keys one after another with the running maximum and sum of the softmax in fp32.
template <typename T, int D>
__global__ void __launch_bounds__(128) attend_prefix_rows_kernel(const vk_prefix_args a) {
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const long long item = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int r = (int)(item / a.Hq), hq = (int)(item % a.Hq), h = hq / (a.Hq / a.KVH);
    if (r >= a.seqs * a.T) return;
    const int own = a.lens[r];
    if (own < 0) return;
    constexpr int E = D / 32;
    float q[E], o[E] = {}, m = -INFINITY, l = 0.f;
    const T* qp = (const T*)a.q + r * a.q_row + hq * a.q_head;
    for (int e = 0; e < E; e++) q[e] = to_f(qp[lane + 32 * e]) * a.scale * 1.4426950408889634f;
    for (int part = 0; part < 2; part++) {
        const int* pages = part ? a.table + (long long)(r / a.T) * a.max_pages : a.prefix_pages;
        const int cap = (part ? a.max_pages : a.max_prefix_pages) * 64;
        int n = part ? own : *a.prefix_len;
        if (n > cap) { vk_set_status(VK_ST_BAD_INDEX); n = cap; }
        for (int i = 0; i < n; i++) {
            int page = pages[i / 64];
            if (page < 0 || page >= a.n_pages) { vk_set_status(VK_ST_BAD_INDEX); page = 0; }
            const long long at = (((long long)page * a.KVH + h) * 64 + i % 64) * D;
            float s = 0.f;
            for (int e = 0; e < E; e++) s += q[e] * to_f(((const T*)a.K)[at + lane + 32 * e]);
            s = warp_sum(s);
            const float mn = fmaxf(m, s), c = mn == -INFINITY ? 1.f : exp2f(m - mn), w = mn == -INFINITY ? 0.f : exp2f(s - mn);
            l = l * c + w;
            for (int e = 0; e < E; e++) o[e] = o[e] * c + w * to_f(((const T*)a.V)[at + lane + 32 * e]);
            m = mn;
        }
    }
    const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
    for (int e = 0; e < E; e++) {
        float v = o[e] * inv;
        if (a.gate) v /= 1.f + expf(-to_f(((const T*)a.gate)[r * a.gate_row + hq * a.gate_head + lane + 32 * e]));
        ((T*)a.out)[r * a.out_row + hq * a.out_head + lane + 32 * e] = from_f<T>(v);
    }
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

}  // namespace

extern "C" {

size_t vk_attend_prefix_workspace_bytes(const vk_prefix_args* a) {
    return prefix_args_ok(a) == VK_OK ? 16 : 0;
}

int vk_attend_prefix(const vk_prefix_args* a, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
    const int ok = prefix_args_ok(a);
    if (ok != VK_OK || a->seqs == 0) return ok;
    if (workspace == nullptr || ((uintptr_t)workspace & 15)) return VK_EINVAL;
    if (workspace_bytes < vk_attend_prefix_workspace_bytes(a)) return VK_ENOSPC;
    const dim3 grid((unsigned)(((long long)a->seqs * a->T * a->Hq + 3) / 4)), block(128);
    if (a->dtype == VK_BF16)
        return (int)(a->D == 128 ? vk_launch(attend_prefix_rows_kernel<__nv_bfloat16, 128>, grid, block, 0, stream, *a)
                                 : vk_launch(attend_prefix_rows_kernel<__nv_bfloat16, 64>, grid, block, 0, stream, *a));
    return (int)(a->D == 128 ? vk_launch(attend_prefix_rows_kernel<__half, 128>, grid, block, 0, stream, *a)
                             : vk_launch(attend_prefix_rows_kernel<__half, 64>, grid, block, 0, stream, *a));
}

}  // extern "C"
