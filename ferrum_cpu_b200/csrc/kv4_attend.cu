// Attention over the cache of 4-bit levels (layout: kv4.cuh): which kernels a call takes.
#include "kv4_ops.cuh"

namespace fc {

int launch_kv4_attend(const Kv4& c, const Kv4Attend& a, const KvRows& rows, int max_rows, int device, cudaStream_t st) {
    const bool step = kv4_step_covers(c, a.group, max_rows);
    // one launch, weights and all, where a cluster holds all columns of a key / value head
    if (step && (!a.mass || max_rows * a.group <= 8)) return launch_kv4_step(c, a, rows, max_rows, nullptr, device, st);
    CallScratch scratch;
    if (a.mass) {
        FC_TRY(scratch.take(device, (size_t)rows.start[c.n_seq] * c.n_kv * a.group * sizeof(float2), st));
        if (!scratch.p) return fail(FC_E_CUDA, "no memory for the softmax statistics of a call that keeps weights");
    }
    float2* const stats = (float2*)scratch.p;
    if (step) {
        FC_TRY(launch_kv4_step(c, a, rows, max_rows, stats, device, st));
    } else {
        if (a.k) FC_TRY(launch_kv4_append(c, a.k, a.v, a.ldkv, rows, max_rows, a.lens, st));
        FC_TRY(launch_kv4_prompt(c, a, rows, max_rows, stats, device, st));
    }
    return a.mass ? launch_kv4_weights(c, a, rows, max_rows, stats, device, st) : FC_OK;
}

}  // namespace fc
