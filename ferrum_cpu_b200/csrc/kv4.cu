// The key / value cache of 4-bit levels: creation, filling, reading back, and eviction by accumulated attention weight. Layout:
// kv4.cuh; attention over it: kv4_attend.cu.
#include <climits>
#include <cmath>

#include "kv4_frag.cuh"

namespace fc {

namespace {

// Rows of k and v into the cache: a warp takes up to four blocks of one row and head, eight lanes a block. Bound: the bytes of long
// prompts, latency of short ones.
__global__ void __launch_bounds__(256) kv4_append_kernel(Kv4 c, const float* __restrict__ k, const float* __restrict__ v, int ldkv, KvRows rows, const int* __restrict__ lens) {
    const int lane = threadIdx.x & 31, seq = blockIdx.z, h = blockIdx.y, first = rows.start[seq], n = rows.start[seq + 1] - first;
    const int len = lens[seq];
    if (len < 0 || len > c.cap - n) return;
    const int warps = gridDim.x * (blockDim.x >> 5), parts = (c.nb + 3) / 4;
    for (int w = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); w < n * parts; w += warps) {
        const int i = w / parts, b = w % parts * 4 + (lane >> 3), pos = len + i, e = lane & 7;
        const bool in = b < c.nb;
        const size_t at = (size_t)(first + i) * ldkv + h * c.dim() + b * kKvBlock + 4 * e, row = c.row(seq, h, pos);
        const float4 none = make_float4(0.0f, 0.0f, 0.0f, 0.0f), kx = in ? *(const float4*)(k + at) : none, vx = in ? *(const float4*)(v + at) : none;
        __half d;
        int level[4];
        quantize4(kx, &d, level);
        const uint32_t word = key_word(level, lane);
        if (in && !(e & 1)) c.kq[row * (c.nb * 4) + (e >> 1) * c.nb + b] = word;
        if (in && !e) c.kd[row * c.nb + b] = d;
        quantize4(vx, &d, level);
        const uint2 half = value_halves(level, lane);
        if (in && e < 2) {
            uint16_t* to = (uint16_t*)c.vq + 2 * ((row >> 1) * (c.nb * 8) + (4 * e) * c.nb + b) + (pos & 1);
            to[0] = (uint16_t)half.x; to[2 * c.nb] = (uint16_t)(half.x >> 16);
            to[4 * c.nb] = (uint16_t)half.y; to[6 * c.nb] = (uint16_t)(half.y >> 16);
        }
        if (in && !e) c.vd[row * c.nb + b] = d;
    }
}

// Positions from[seq] .. + n of every sequence as the values that they stand for: out [n_seq][n][n_kv][dim], zeros outside the cache.
__global__ void kv4_read_kernel(Kv4 c, const int* __restrict__ from, int n, float* __restrict__ k, float* __restrict__ v) {
    const int dim = c.dim(), seq = blockIdx.y, base = from ? from[seq] : 0;
    const size_t all = (size_t)n * c.n_kv * dim;
    for (size_t e = (size_t)blockIdx.x * blockDim.x + threadIdx.x; e < all; e += (size_t)gridDim.x * blockDim.x) {
        const int ch = (int)(e % dim), h = (int)(e / dim % c.n_kv), i = (int)(e / dim / c.n_kv);
        const long long pos = (long long)base + i;
        float kx = 0.0f, vx = 0.0f;
        if (pos >= 0 && pos < c.cap) {
            const int b = ch / 32, r = ch % 32;
            const size_t row = c.row(seq, h, (int)pos), pair = c.row(seq, h, (int)pos & ~1) >> 1;
            const unsigned kw = c.kq[row * (c.nb * 4) + (r >> 3) * c.nb + b];
            const unsigned vw = ((const uint16_t*)c.vq)[2 * (pair * (c.nb * 8) + (r & 7) * c.nb + b) + (pos & 1)];
            kx = __half2float(c.kd[row * c.nb + b]) * (float)((int)(kw >> (4 * (r & 7)) & 15) - 8);
            vx = __half2float(c.vd[row * c.nb + b]) * (float)((int)(vw >> (4 * (r >> 3)) & 15) - 8);
        }
        k[(size_t)seq * all + e] = kx;
        v[(size_t)seq * all + e] = vx;
    }
}

// Weights in their order as unsigned keys; NaN is the least.
__device__ __forceinline__ unsigned weight_key(float w) {
    w += 0.0f;                                     // -0 is 0
    const unsigned b = __float_as_uint(w);
    return w != w ? 0u : b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}

constexpr int ET = 512;

// One CTA a (sequence, head): the key of the last position that is kept by bisection, then the kept positions in order.
__global__ void __launch_bounds__(ET) kv4_evict_kernel(Kv4 src, Kv4 dst, const int* __restrict__ lens, int* __restrict__ lens_out, int budget, int recent,
                                                       const float* __restrict__ mass, float* __restrict__ mass_out, int* __restrict__ kept) {
    __shared__ int found[ET / 32], base_more, base_tie;
    const int tid = threadIdx.x, h = blockIdx.x, seq = blockIdx.y, head = seq * src.n_kv + h;
    int len = lens[seq];
    len = len < 0 ? 0 : min(len, src.cap);
    const int left = min(len, budget);
    if (tid == 0 && h == 0) lens_out[seq] = left;
    const float* m = mass + (size_t)head * src.cap;
    const bool all = len <= budget;
    const int old = all ? len : len - recent, want = all ? old : budget - recent;
    auto count = [&](unsigned at) {
        int n = 0;
        for (int j = tid; j < old; j += ET) n += weight_key(m[j]) >= at;
        for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
        __syncthreads();
        if ((tid & 31) == 0) found[tid >> 5] = n;
        __syncthreads();
        n = 0;
        for (int w = 0; w < ET / 32; ++w) n += found[w];
        return n;
    };
    unsigned cut = 0;
    for (int bit = 31; bit >= 0 && !all; --bit)
        if (count(cut | (1u << bit)) >= want) cut |= 1u << bit;
    const int more = all ? 0 : cut == 0xffffffffu ? 0 : count(cut + 1), ties = want - more;
    if (tid == 0) base_more = base_tie = 0;
    __syncthreads();
    for (int j0 = 0; j0 < len; j0 += ET) {
        const int j = j0 + tid;
        const unsigned key = j < old ? weight_key(m[j]) : 0u;
        const bool sure = j < len && (all || j >= old || (want > 0 && key > cut)), tie = !all && want > 0 && j < old && key == cut;
        // how many of either kind come before j
        const unsigned ms = __ballot_sync(0xffffffffu, sure), mt = __ballot_sync(0xffffffffu, tie), below = (1u << (tid & 31)) - 1;
        __syncthreads();
        if ((tid & 31) == 0) found[tid >> 5] = __popc(ms) | __popc(mt) << 16;
        __syncthreads();
        int s = base_more + __popc(ms & below), t = base_tie + __popc(mt & below), all_s = 0, all_t = 0;
        for (int w = 0; w < ET / 32; ++w) {
            if (w < (tid >> 5)) { s += found[w] & 0xffff; t += found[w] >> 16; }
            all_s += found[w] & 0xffff; all_t += found[w] >> 16;
        }
        if (sure || (tie && t < ties)) {
            const int to = s + min(t, ties);
            const size_t a = src.row(seq, h, j), b = dst.row(seq, h, to);
            for (int w = 0; w < src.nb * 4; ++w) dst.kq[b * (src.nb * 4) + w] = src.kq[a * (src.nb * 4) + w];
            const uint16_t* va = (const uint16_t*)src.vq + (a >> 1) * (src.nb * 16) + (a & 1);
            uint16_t* vb = (uint16_t*)dst.vq + (b >> 1) * (src.nb * 16) + (b & 1);
            for (int w = 0; w < src.nb * 8; ++w) vb[2 * w] = va[2 * w];
            for (int w = 0; w < src.nb; ++w) { dst.kd[b * src.nb + w] = src.kd[a * src.nb + w]; dst.vd[b * src.nb + w] = src.vd[a * src.nb + w]; }
            if (mass_out) mass_out[(size_t)head * dst.cap + to] = m[j];
            if (kept) kept[(size_t)head * budget + to] = j;
        }
        __syncthreads();
        if (tid == 0) { base_more += all_s; base_tie += all_t; }
        __syncthreads();
    }
    for (int j = left + tid; kept && j < budget; j += ET) kept[(size_t)head * budget + j] = -1;
}

}  // namespace

int launch_kv4_append(const Kv4& c, const float* k, const float* v, int ldkv, const KvRows& rows, int max_rows, const int* lens, cudaStream_t st) {
    const long long warps = (long long)max_rows * ((c.nb + 3) / 4);
    const dim3 grid((unsigned)std::min<long long>((warps + 7) / 8, 4096), c.n_kv, c.n_seq);
    kv4_append_kernel<<<grid, 256, 0, st>>>(c, k, v, ldkv, rows, lens);
    FC_LAUNCHED();
    return FC_OK;
}

int make_device(int device) {
    // asking is cheaper than setting, and nearly every call finds its device current
    int current = -1;
    FC_CUDA(cudaGetDevice(&current));
    if (current != device) FC_CUDA(cudaSetDevice(device));
    return FC_OK;
}

// The rows each sequence brings, as their places among the packed rows. counts null: one each.
static int kv4_rows(const fc_kv4* c, const int32_t* counts, const char* what, KvRows* rows, int* max_rows) {
    long long at = 0;
    *max_rows = 0;
    for (int s = 0; s < c->c.n_seq; ++s) {
        const int n = counts ? counts[s] : 1;
        if (n < 0) return fail(FC_E_SHAPE, "%s: sequence %d has %d rows", what, s, n);
        if (n > c->c.cap) return fail(FC_E_DIM, "%s: %d rows of sequence %d do not fit a cache of %d positions", what, n, s, c->c.cap);
        rows->start[s] = (int)at;
        at += n;
        if (at > INT_MAX) return fail(FC_E_SHAPE, "%s: more than %d rows", what, INT_MAX);
        if (n > *max_rows) *max_rows = n;
    }
    rows->start[c->c.n_seq] = (int)at;
    return FC_OK;
}

}  // namespace fc

using namespace fc;

extern "C" {

int fc_kv4_create(int device, int n_seq, int n_kv_head, int head_dim, int capacity, fc_kv4** out) {
    if (!out) return fail(FC_E_ARG, "fc_kv4_create: null argument");
    *out = nullptr;
    if (n_seq <= 0 || n_seq > kKvMaxSeq || n_kv_head <= 0 || n_kv_head > 65535 || capacity <= 0 || capacity > (1 << 24))
        return fail(FC_E_SHAPE, "fc_kv4_create: %d sequences (1..%d), %d heads, %d positions (1..2^24)", n_seq, kKvMaxSeq, n_kv_head, capacity);
    if (head_dim <= 0 || head_dim % kKvBlock || head_dim > 256)
        return fail(FC_E_SHAPE, "fc_kv4_create: head_dim %d must be a multiple of %d, at most 256", head_dim, kKvBlock);
    FC_TRY(select_device(device));
    FC_TRY(scratch_retain(device));
    fc_kv4* c = new fc_kv4();
    c->device = device;
    auto build = [&]() -> int {
        const int pad = (capacity + kKvTile - 1) / kKvTile * kKvTile;
        const size_t rows = (size_t)n_seq * n_kv_head * pad, q = rows * head_dim / 2, d = rows * (head_dim / kKvBlock) * 2;
        c->c = Kv4{nullptr, nullptr, nullptr, nullptr, n_seq, n_kv_head, head_dim / kKvBlock, capacity, pad};
        FC_TRY(c->arena.alloc((void**)&c->c.kq, q));
        FC_TRY(c->arena.alloc((void**)&c->c.vq, q));
        FC_TRY(c->arena.alloc((void**)&c->c.kd, d));
        FC_TRY(c->arena.alloc((void**)&c->c.vd, d));
        FC_CUDA(cudaMemset(c->c.kq, 0, q));
        FC_CUDA(cudaMemset(c->c.vq, 0, q));
        FC_CUDA(cudaMemset(c->c.kd, 0, d));
        FC_CUDA(cudaMemset(c->c.vd, 0, d));
        FC_CUDA(cudaDeviceSynchronize());
        return FC_OK;
    };
    const int rc = build();
    if (rc != FC_OK) { fc_kv4_free(c); return rc; }
    *out = c;
    return FC_OK;
}

void fc_kv4_free(fc_kv4* c) {
    if (!c) return;
    cudaSetDevice(c->device);
    cudaDeviceSynchronize();
    c->arena.release();
    scratch_release(c->device);
    delete c;
}

int fc_kv4_append_dev(fc_kv4* c, const float* k, const float* v, int ldkv, const int32_t* rows, const int32_t* lens, void* stream) {
    if (!c || !k || !v || !lens) return fail(FC_E_ARG, "fc_kv4_append_dev: null argument");
    if (!aligned16(k) || !aligned16(v)) return fail(FC_E_ARG, "fc_kv4_append_dev: k and v must be 16-byte aligned");
    if (ldkv % 4 || ldkv < c->c.n_kv * c->c.dim()) return fail(FC_E_SHAPE, "fc_kv4_append_dev: ldkv %d must be a multiple of 4, at least %d", ldkv, c->c.n_kv * c->c.dim());
    KvRows r;
    int most = 0;
    FC_TRY(kv4_rows(c, rows, "fc_kv4_append_dev", &r, &most));
    if (!most) return FC_OK;
    FC_TRY(make_device(c->device));
    return launch_kv4_append(c->c, k, v, ldkv, r, most, lens, (cudaStream_t)stream);
}

int fc_kv4_attend_dev(fc_kv4* c, const float* q, int ldq, int n_head, const float* k, const float* v, int ldkv, const int32_t* rows,
                      const int32_t* lens, float scale, float* mass, float* out, int ldo, void* stream) {
    if (!c || !q || !lens || !out || !k != !v) return fail(FC_E_ARG, "fc_kv4_attend_dev: null argument");
    const int dim = c->c.dim();
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out))
        return fail(FC_E_ARG, "fc_kv4_attend_dev: q, k, v and out must be 16-byte aligned");
    if (n_head <= 0 || n_head % c->c.n_kv) return fail(FC_E_DIM, "fc_kv4_attend_dev: n_head %d must be a multiple of the cache's %d key / value heads", n_head, c->c.n_kv);
    if (n_head > 65535 || ldq % 4 || ldo % 4 || ldq < n_head * dim || ldo < n_head * dim)
        return fail(FC_E_SHAPE, "fc_kv4_attend_dev: ldq %d and ldo %d must be multiples of 4, at least n_head %d x %d", ldq, ldo, n_head, dim);
    if (k && (ldkv % 4 || ldkv < c->c.n_kv * dim)) return fail(FC_E_SHAPE, "fc_kv4_attend_dev: ldkv %d must be a multiple of 4, at least %d", ldkv, c->c.n_kv * dim);
    if (!std::isfinite(scale)) return fail(FC_E_ARG, "fc_kv4_attend_dev: scale must be finite");
    KvRows r;
    int most = 0;
    FC_TRY(kv4_rows(c, rows, "fc_kv4_attend_dev", &r, &most));
    if (!most) return FC_OK;
    if ((long long)most * (n_head / c->c.n_kv) > INT_MAX / 2) return fail(FC_E_SHAPE, "fc_kv4_attend_dev: %d rows of %d heads", most, n_head);
    FC_TRY(make_device(c->device));
    const Kv4Attend a = {q, k, v, out, ldq, ldkv, ldo, n_head / c->c.n_kv, scale != 0.0f ? scale : 1.0f / sqrtf((float)dim), lens, mass};
    return launch_kv4_attend(c->c, a, r, most, c->device, (cudaStream_t)stream);
}

int fc_kv4_read_dev(const fc_kv4* c, const int32_t* from, int n, float* k, float* v, void* stream) {
    if (!c || !k || !v) return fail(FC_E_ARG, "fc_kv4_read_dev: null argument");
    if (n < 0) return fail(FC_E_SHAPE, "fc_kv4_read_dev: n = %d", n);
    if (!n) return FC_OK;
    FC_TRY(make_device(c->device));
    const size_t all = (size_t)n * c->c.n_kv * c->c.dim();
    const dim3 grid((unsigned)std::min<size_t>((all + 255) / 256, 148 * 16), c->c.n_seq);
    kv4_read_kernel<<<grid, 256, 0, (cudaStream_t)stream>>>(c->c, from, n, k, v);
    FC_LAUNCHED();
    return FC_OK;
}

int fc_kv4_evict_dev(const fc_kv4* src, fc_kv4* dst, const int32_t* lens, int32_t* lens_out, int budget, int recent, const float* mass,
                     float* mass_out, int32_t* kept, void* stream) {
    if (!src || !dst || !lens || !lens_out || !mass) return fail(FC_E_ARG, "fc_kv4_evict_dev: null argument");
    if (src == dst || mass == mass_out || lens == lens_out) return fail(FC_E_ARG, "fc_kv4_evict_dev: what is left goes to a cache, weights and lengths of its own");
    const Kv4 &a = src->c, &b = dst->c;
    if (src->device != dst->device || a.n_seq != b.n_seq || a.n_kv != b.n_kv || a.nb != b.nb)
        return fail(FC_E_DIM, "fc_kv4_evict_dev: the caches differ in device, sequences, heads or head_dim");
    if (budget <= 0 || recent < 0 || recent > budget) return fail(FC_E_SHAPE, "fc_kv4_evict_dev: budget %d, recent %d", budget, recent);
    if (budget > b.cap) return fail(FC_E_DIM, "fc_kv4_evict_dev: a budget of %d does not fit %d positions", budget, b.cap);
    FC_TRY(make_device(src->device));
    kv4_evict_kernel<<<dim3(a.n_kv, a.n_seq), ET, 0, (cudaStream_t)stream>>>(a, b, lens, lens_out, budget, recent, mass, mass_out, kept);
    FC_LAUNCHED();
    return FC_OK;
}

}  // extern "C"
