// Attention over the cache of 4-bit levels (layout: kv4.cuh): out = softmax(scale q K^T) V, where row i of a sequence's n new rows sees
// the positions up to its own.
#include "kv4_ops.cuh"

namespace fc {

namespace {

constexpr int AT = 256, CHUNK = 1024;

__device__ __forceinline__ float key_at(const Kv4& c, size_t row, int ch) {
    const int b = ch / 32, r = ch % 32;
    const unsigned w = c.kq[row * (c.nb * 4) + (r >> 3) * c.nb + b];
    return __half2float(c.kd[row * c.nb + b]) * (float)((int)(w >> (4 * (r & 7)) & 15) - 8);
}
__device__ __forceinline__ float value_at(const Kv4& c, size_t row, int ch) {
    const int b = ch / 32, r = ch % 32;
    const unsigned w = ((const uint16_t*)c.vq)[2 * ((row >> 1) * (c.nb * 8) + (r & 7) * c.nb + b) + (row & 1)];
    return __half2float(c.vd[row * c.nb + b]) * (float)((int)(w >> (4 * (r >> 3)) & 15) - 8);
}

// How many positions row i of n sees; negative: the sequence's length is none.
__device__ __forceinline__ int seen_by(const Kv4& c, const Kv4Attend& a, int seq, int n, int i) {
    const int len = a.lens[seq];
    if (a.k) return len < 0 || len > c.cap - n ? -1 : len + i + 1;
    return len < 0 || len > c.cap ? -1 : max(0, len - n + i + 1);
}

// One CTA a (row, query head): scores of CHUNK positions in shared memory, a running maximum and sum, a thread per channel.
__global__ void __launch_bounds__(AT) kv4_attend_kernel(Kv4 c, Kv4Attend a, KvRows rows, float2* __restrict__ stats) {
    __shared__ float qs[256], s[CHUNK], red[AT / 32], acc[AT];
    const int tid = threadIdx.x, dim = c.dim(), head = blockIdx.y, seq = blockIdx.z, h = head / a.group;
    const int first = rows.start[seq], n = rows.start[seq + 1] - first;
    for (int i = blockIdx.x; i < n; i += gridDim.x) {
        const int seen = seen_by(c, a, seq, n, i);
        float* out = a.out + (size_t)(first + i) * a.ldo + head * dim;
        if (seen < 0) {
            for (int ch = tid; ch < dim; ch += AT) out[ch] = __int_as_float(0x7fffffff);
            continue;
        }
        __syncthreads();
        for (int ch = tid; ch < dim; ch += AT) qs[ch] = a.q[(size_t)(first + i) * a.ldq + head * dim + ch] * a.scale;
        float m = -INFINITY, l = 0.0f, o = 0.0f;
        const int ch = tid % dim, part = tid / dim, parts = AT / dim;
        for (int j0 = 0; j0 < seen; j0 += CHUNK) {
            const int jn = min(CHUNK, seen - j0);
            __syncthreads();
            float top = -INFINITY;
            for (int j = tid; j < jn; j += AT) {
                const size_t row = c.row(seq, h, j0 + j);
                float x = 0.0f;
                for (int e = 0; e < dim; ++e) x += qs[e] * key_at(c, row, e);
                s[j] = x;
                top = fmaxf(top, x);
            }
            for (int w = 16; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
            if ((tid & 31) == 0) red[tid >> 5] = top;
            __syncthreads();
            top = m;
            for (int w = 0; w < AT / 32; ++w) top = fmaxf(top, red[w]);
            const float back = expf(m - top);
            m = top;
            o *= back;
            l *= back;
            __syncthreads();
            for (int j = tid; j < jn; j += AT) s[j] = expf(s[j] - m);
            __syncthreads();
            for (int j = 0; j < jn; ++j) l += s[j];
            if (part < parts)
                for (int j = part; j < jn; j += parts) o += s[j] * value_at(c, c.row(seq, h, j0 + j), ch);
        }
        acc[tid] = o;
        __syncthreads();
        if (tid < dim) {
            o = 0.0f;
            for (int p = 0; p < parts; ++p) o += acc[p * dim + tid];
            out[tid] = seen > 0 ? o / l : 0.0f;
        }
        if (tid == 0 && stats) stats[((size_t)first + i) * (c.n_kv * a.group) + head] = make_float2(m, l);
    }
}

// The weights that a position receives, over the rows that see it and the heads that share it. One warp a position.
__global__ void __launch_bounds__(AT) kv4_mass_kernel(Kv4 c, Kv4Attend a, KvRows rows, const float2* __restrict__ stats) {
    const int lane = threadIdx.x & 31, h = blockIdx.y, seq = blockIdx.z, dim = c.dim();
    const int first = rows.start[seq], n = rows.start[seq + 1] - first;
    const int all = n ? seen_by(c, a, seq, n, n - 1) : 0, old = a.k ? a.lens[seq] : all;
    for (int j = blockIdx.x * (AT / 32) + (threadIdx.x >> 5); j < all; j += gridDim.x * (AT / 32)) {
        const size_t row = c.row(seq, h, j);
        float sum = 0.0f;
        for (int i = 0; i < n; ++i) {
            if (seen_by(c, a, seq, n, i) <= j) continue;
            for (int g = 0; g < a.group; ++g) {
                const int head = h * a.group + g;
                const float* q = a.q + (size_t)(first + i) * a.ldq + head * dim;
                float x = 0.0f;
                for (int e = lane; e < dim; e += 32) x += q[e] * a.scale * key_at(c, row, e);
                for (int w = 16; w > 0; w >>= 1) x += __shfl_xor_sync(0xffffffffu, x, w);
                const float2 st = stats[((size_t)first + i) * (c.n_kv * a.group) + head];
                sum += expf(x - st.x) / st.y;
            }
        }
        float* m = a.mass + ((size_t)seq * c.n_kv + h) * c.cap + j;
        if (lane == 0) *m = (j < old ? *m : 0.0f) + sum;
    }
}

}  // namespace

int launch_kv4_attend(const Kv4& c, const Kv4Attend& a, const KvRows& rows, int max_rows, int device, cudaStream_t st) {
    const bool step = kv4_step_covers(c, a.group, max_rows);
    if (step && (!a.mass || max_rows * a.group <= 8)) return launch_kv4_step(c, a, rows, max_rows, nullptr, device, st);
    if (a.k) FC_TRY(launch_kv4_append(c, a.k, a.v, a.ldkv, rows, max_rows, a.lens, st));
    CallScratch scratch;
    const int heads = c.n_kv * a.group;
    if (a.mass) {
        FC_TRY(scratch.take(device, (size_t)rows.start[c.n_seq] * heads * sizeof(float2), st));
        if (!scratch.p) return fail(FC_E_CUDA, "no memory for the softmax statistics of a call that keeps weights");
    }
    kv4_attend_kernel<<<dim3(std::min(max_rows, 1024), heads, c.n_seq), AT, 0, st>>>(c, a, rows, (float2*)scratch.p);
    FC_LAUNCHED();
    if (a.mass) {
        kv4_mass_kernel<<<dim3(std::min((c.cap + 7) / 8, 1024), c.n_kv, c.n_seq), AT, 0, st>>>(c, a, rows, (const float2*)scratch.p);
        FC_LAUNCHED();
    }
    return FC_OK;
}

}  // namespace fc
