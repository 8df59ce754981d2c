// Launchers of the 4-bit cache's kernels (kv4.cu, kv4_attend.cu).
#pragma once
#include <algorithm>

#include "kv4.cuh"

namespace fc {

struct Kv4Attend {
    const float *q, *k, *v;      // k, v: the call's new rows, or null
    float* out;
    int ldq, ldkv, ldo;
    int group;                   // query heads a key / value head
    float scale;
    const int* lens;             // positions before the call (k, v given) or with the call's rows
    float* mass;                 // [n_seq][n_kv][cap] or null
};

// A zeroed cache in the arena's memory.
int kv4_make(Arena& arena, int n_seq, int n_kv, int dim, int cap, Kv4* c);
// state (may be null): with a stream that is done or in error all of it moves, into a dst of the same capacity.
int launch_kv4_evict(const Kv4& src, const Kv4& dst, const int* lens, int* lens_out, int budget, int recent, const float* mass, float* mass_out, int* kept,
                     int device, cudaStream_t st, const StepState* state = nullptr);
int make_device(int device);
int launch_kv4_append(const Kv4& c, const float* k, const float* v, int ldkv, const KvRows& rows, int max_rows, const int* lens, cudaStream_t st);
// kv4_step.cu: few query rows a key / value head; stats: where a row's maximum (base 2) and sum go, if another kernel adds up its weights.
bool kv4_step_covers(const Kv4& c, int group, int max_rows);
int launch_kv4_step(const Kv4& c, const Kv4Attend& a, const KvRows& rows, int max_rows, float2* stats, int device, cudaStream_t st);
// kv4_prompt.cu: any number of them; and the weights that the positions receive, from such statistics.
int launch_kv4_prompt(const Kv4& c, const Kv4Attend& a, const KvRows& rows, int max_rows, float2* stats, int device, cudaStream_t st);
int launch_kv4_weights(const Kv4& c, const Kv4Attend& a, const KvRows& rows, int max_rows, const float2* stats, int device, cudaStream_t st);
int launch_kv4_attend(const Kv4& c, const Kv4Attend& a, const KvRows& rows, int max_rows, int device, cudaStream_t st);

}  // namespace fc
