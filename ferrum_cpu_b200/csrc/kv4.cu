// The key / value cache of 4-bit levels: creation, filling, reading back, and eviction by accumulated attention weight. Layout:
// kv4.cuh; attention over it: kv4_attend.cu.
#include <climits>
#include <cmath>

#include "kv4_frag.cuh"

namespace fc {

namespace {

// Rows of k and v into the cache: a warp takes up to four blocks of one row and head, eight lanes a block, keys and then values. Bound: for
// long rows the instructions of the rounding (2 x 131 million values in 420 us, 2.5 TB/s of f32 read; keys and values by warps of their
// own: 550), for short ones latency.
__global__ void __launch_bounds__(256) kv4_append_kernel(Kv4 c, const float* __restrict__ k, const float* __restrict__ v, int ldkv, KvRows rows, const int* __restrict__ lens) {
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31, seq = blockIdx.z, h = blockIdx.y, first = rows.start[seq], n = rows.start[seq + 1] - first;
    const int len = lens[seq];
    if (len < 0 || len > c.cap - n) return;
    const int warps = gridDim.x * (blockDim.x >> 5), two = c.nb > 4;         // pieces a row: one, or two
    for (int w = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); w < n << two; w += warps) {
        const int i = w >> two, b = (w & two) * 4 + (lane >> 3), pos = len + i, e = lane & 7;
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

// Positions from[seq] .. + n of every sequence as the values that they stand for: out [n_seq][n][n_kv][dim], zeros outside the cache. A thread
// writes eight channels of a row, of keys from one word, of values from the nibble j of eight half words. Bound: the bytes written (134 MB in 27 us, 4.9 TB/s; a fill of as much
// takes 21; 32 us without the streaming hint, 39 with each lane's 32 bytes stored by itself).
__global__ void __launch_bounds__(256) kv4_read_kernel(Kv4 c, const int* __restrict__ from, int n, float* __restrict__ k, float* __restrict__ v) {
    pdl_trigger();
    pdl_wait();
    const int parts = c.nb * 4, seq = blockIdx.y, base = from ? from[seq] : 0;
    const int per = 128 / parts, e = threadIdx.x & 127, part = e % parts, b = part >> 2, t = part & 3;      // rows a block: half of it keys, half values
    const bool values = threadIdx.x >= 128;
    if (e >= per * parts) return;
    // rows of all heads in the order in which they are written
    const unsigned first = blockIdx.x * per + e / parts, stride = gridDim.x * per, step_i = stride / (unsigned)c.n_kv, step_h = stride % (unsigned)c.n_kv;
    long long i = first / (unsigned)c.n_kv;
    int h = (int)(first % (unsigned)c.n_kv);
    for (; i < n; i += step_i, h += step_h) {
        if (h >= c.n_kv) {
            h -= c.n_kv;
            if (++i >= n) break;
        }
        const long long pos = base + i;
        float x[8] = {};
        if (pos >= 0 && pos < c.cap) {
            const size_t row = c.row(seq, h, (int)pos);
            if (values) {
                const uint16_t* w = (const uint16_t*)c.vq + 2 * ((row >> 1) * (c.nb * 8) + b) + (pos & 1);
                const float d = __half2float(c.vd[row * c.nb + b]);
#pragma unroll
                for (int g = 0; g < 8; ++g) x[g] = d * (float)((int)(w[2 * g * c.nb] >> (4 * t) & 15) - 8);
            } else {
                const uint32_t w = c.kq[row * (c.nb * 4) + t * c.nb + b];
                const float d = __half2float(c.kd[row * c.nb + b]);
#pragma unroll
                for (int g = 0; g < 8; ++g) x[g] = d * (float)((int)(w >> (4 * g) & 15) - 8);
            }
        }
        // two lanes exchange halves, so that a store writes whole lines: the even lane's channels first, then the odd one's
        const bool odd = threadIdx.x & 1;
        float y[4];
#pragma unroll
        for (int g = 0; g < 4; ++g) y[g] = __shfl_xor_sync(3u << (threadIdx.x & 30), odd ? x[g] : x[4 + g], 1);
        float4* to = (float4*)((values ? v : k) + ((((size_t)seq * n + i) * c.n_kv + h) * parts + (part & ~1)) * 8) + odd;
        __stcs(to, odd ? make_float4(y[0], y[1], y[2], y[3]) : make_float4(x[0], x[1], x[2], x[3]));
        __stcs(to + 2, odd ? make_float4(x[4], x[5], x[6], x[7]) : make_float4(y[0], y[1], y[2], y[3]));
    }
}

// Weights in their order as unsigned keys; NaN is the least.
__device__ __forceinline__ unsigned weight_key(float w) {
    w += 0.0f;                                     // -0 is 0
    const unsigned b = __float_as_uint(w);
    return w != w ? 0u : b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}

// (positions above KEYS have their weights read from memory in each pass, from L2 mostly: 64 heads of 128 to 2048 positions, from 16384 25.5 us, 17500 23.5,
// 30000 33.7)
constexpr int ET = 1024, BINS = 2048, KEYS = 16384, LISTED = 2048;
struct __align__(16) EvictShared {
    unsigned key[KEYS];
    unsigned bins[BINS];
    int src[LISTED];                               // where the rows of a window of dst come from
    int warp_n[ET / 32], warp_t[ET / 32];
    int digit, above, in_bin, listed;
};

// What stays of a (sequence, head), shared by gridDim.x CTAs. Each finds the key of the last position that stays for itself (three passes
// of 11, 11 and 10 bits over the keys, in shared memory where they fit): the row of weights is short next to what is moved, and no CTA has to
// wait for another. Then each brings a range of dst's rows. Bound: latency, and the bytes moved of long caches (64 heads of 128, 16001 to
// 2048 positions: 25 us, 13 of them for the move of 38 MB).
__global__ void __launch_bounds__(ET, 1) kv4_evict_kernel(Kv4 src, Kv4 dst, const int* __restrict__ lens, int* __restrict__ lens_out, int budget, int recent,
                                                          const float* __restrict__ mass, float* __restrict__ mass_out, int* __restrict__ kept,
                                                          const StepState* state) {
    extern __shared__ __align__(16) char raw[];
    EvictShared& s = *(EvictShared*)raw;
    pdl_trigger();
    pdl_wait();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, h = blockIdx.y, seq = blockIdx.z, head = seq * src.n_kv + h;
    int len = lens[seq];
    len = len < 0 ? 0 : min(len, src.cap);
    if (state && (state->done | state->error)) budget = dst.cap;
    const int left = min(len, budget);
    if (tid == 0 && h == 0 && blockIdx.x == 0) lens_out[seq] = left;
    // this CTA's rows of dst, an even number from an even one on
    const int share = ((left + (int)gridDim.x - 1) / (int)gridDim.x + 1) & ~1, d0 = min(left, (int)blockIdx.x * share), d1 = min(left, d0 + share);
    for (int j = max(left, (int)blockIdx.x * ((budget + (int)gridDim.x - 1) / (int)gridDim.x)) + tid; kept && j < min(budget, ((int)blockIdx.x + 1) * ((budget + (int)gridDim.x - 1) / (int)gridDim.x)); j += ET)
        kept[(size_t)head * budget + j] = -1;
    if (d0 >= d1) return;
    const float* m = mass + (size_t)head * src.cap;
    const bool all = len <= budget;
    const int old = all ? 0 : len - recent, want = budget - recent;      // of the first `old` positions the `want` heaviest
    const bool fits = old <= KEYS;
    if (fits)
#pragma unroll 16
        for (int j = tid; j < old; j += ET) s.key[j] = weight_key(__ldg(m + j));
    auto key = [&](int j) { return fits ? s.key[j] : weight_key(__ldg(m + j)); };
    unsigned cut = 0;
    int ties = want;                               // how many of those at the cut stay, the first ones
    if (!all && want > 0) {
        int shift = 21, width = 11, listed = 0;
        unsigned* const list = (unsigned*)s.src;
        for (int pass = 0; pass < 3; ++pass) {
            for (int b = tid; b < BINS; b += ET) s.bins[b] = 0;
            if (tid == 0) s.listed = 0;
            __syncthreads();
            const unsigned high = pass ? cut >> (shift + width) : 0, mask = (1u << width) - 1;
            if (pass == 0) {
#pragma unroll 8
                for (int j = tid; j < old; j += ET) atomicAdd(&s.bins[key(j) >> shift], 1u);
            } else if (pass == 1) {
                // the keys of the first digit's bin, listed where they fit
                const bool list_them = s.in_bin <= LISTED;
#pragma unroll 4
                for (int j = tid; j < old; j += ET) {
                    const unsigned k = key(j);
                    if (k >> (shift + width) != high) continue;
                    atomicAdd(&s.bins[k >> shift & mask], 1u);
                    if (list_them) list[atomicAdd(&s.listed, 1)] = k;
                }
                listed = list_them;
            } else if (listed) {
                for (int j = tid; j < s.in_bin; j += ET)
                    if (list[j] >> (shift + width) == high) atomicAdd(&s.bins[list[j] >> shift & mask], 1u);
            } else {
#pragma unroll 4
                for (int j = tid; j < old; j += ET) {
                    const unsigned k = key(j);
                    if (k >> (shift + width) == high) atomicAdd(&s.bins[k >> shift & mask], 1u);
                }
            }
            __syncthreads();
            // from the largest digit down: EACH a thread
            constexpr int EACH = BINS / ET;
            int n[EACH], sum = 0;
#pragma unroll
            for (int i = 0; i < EACH; ++i) { n[i] = (int)s.bins[BINS - 1 - (EACH * tid + i)]; sum += n[i]; }
            int incl = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += x;
            }
            if (lane == 31) s.warp_n[warp] = incl;
            __syncthreads();
            int before = incl - sum;
            for (int w = 0; w < warp; ++w) before += s.warp_n[w];
#pragma unroll
            for (int i = 0; i < EACH; ++i) {
                if (before < ties && before + n[i] >= ties) {
                    s.digit = BINS - 1 - (EACH * tid + i);
                    s.above = before;
                    if (pass == 0) s.in_bin = n[i];
                }
                before += n[i];
            }
            __syncthreads();
            cut |= (unsigned)s.digit << shift;
            ties -= s.above;
            width = pass == 1 ? 10 : 11;
            shift -= width;
            if (shift < 0) shift = 0;
        }
    }
    __syncthreads();
    // thread t walks positions [t * per, ..) (an odd stride meets every bank): how many of them are sure to stay, and how many are at the cut
    const int per = ((old + ET - 1) / ET) | 1, j0 = min(old, tid * per), j1 = min(old, j0 + per);
    int sure = 0, tie = 0;
    if (want > 0)
#pragma unroll 8
        for (int j = j0; j < j1; ++j) {
            const unsigned k = key(j);
            sure += k > cut;
            tie += k == cut;
        }
    int is = sure, it = tie;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int a = __shfl_up_sync(0xffffffffu, is, o), b = __shfl_up_sync(0xffffffffu, it, o);
        if (lane >= o) { is += a; it += b; }
    }
    if (lane == 31) { s.warp_n[warp] = is; s.warp_t[warp] = it; }
    __syncthreads();
    int s0 = is - sure, t0 = it - tie;
    for (int w = 0; w < warp; ++w) { s0 += s.warp_n[w]; t0 += s.warp_t[w]; }
    const int first = s0 + min(t0, ties), last = s0 + sure + min(t0 + tie, ties);    // this thread's rows of dst
    const size_t da = dst.row(seq, h, 0), sa = src.row(seq, h, 0);
    const int nb = src.nb;
    for (int w0 = d0; w0 < d1; w0 += LISTED) {
        const int w1 = min(d1, w0 + LISTED), rows = w1 - w0;
        __syncthreads();
        if (!all && want > 0 && first < w1 && last > w0) {
            int to = first, t = t0;
            for (int j = j0; j < j1; ++j) {
                const unsigned k = key(j);
                if (k > cut || (k == cut && t++ < ties)) {
                    if (to >= w0 && to < w1) s.src[to - w0] = j;
                    ++to;
                }
            }
        }
        // the recent ones, or all
        const int body = all ? 0 : want;
        for (int to = max(w0, body) + tid; to < w1; to += ET) s.src[to - w0] = all ? to : to - body + old;
        __syncthreads();
#pragma unroll 4
        for (int e = tid; e < rows * nb; e += ET) {
            const int i = e / nb, q = e % nb;
            ((uint4*)(dst.kq + (da + w0 + i) * (nb * 4)))[q] = __ldg((const uint4*)(src.kq + (sa + s.src[i]) * (nb * 4)) + q);
        }
        const int pairs = rows >> 1;
#pragma unroll 4
        for (int e = tid; e < pairs * 2 * nb; e += ET) {
            const int i = e / (2 * nb), q = e % (2 * nb), a = s.src[2 * i], b = s.src[2 * i + 1];
            const uint4 x = __ldg((const uint4*)(src.vq + ((sa + a) >> 1) * (nb * 8)) + q), y = __ldg((const uint4*)(src.vq + ((sa + b) >> 1) * (nb * 8)) + q);
            const unsigned pick = (a & 1 ? 0x32 : 0x10) | (b & 1 ? 0x7600 : 0x5400);
            ((uint4*)(dst.vq + ((da + w0) / 2 + i) * (nb * 8)))[q] =
                make_uint4(__byte_perm(x.x, y.x, pick), __byte_perm(x.y, y.y, pick), __byte_perm(x.z, y.z, pick), __byte_perm(x.w, y.w, pick));
        }
        if (rows & 1) {                            // a last row alone: what lies behind it stays as it was
            const int a = s.src[rows - 1];
            const uint16_t* x = (const uint16_t*)(src.vq + ((sa + a) >> 1) * (nb * 8)) + (a & 1);
            uint16_t* y = (uint16_t*)(dst.vq + ((da + w1 - 1) / 2) * (nb * 8));
            for (int e = tid; e < 8 * nb; e += ET) y[2 * e] = x[2 * e];
        }
#pragma unroll 4
        for (int e = tid; e < rows * nb; e += ET) {
            const int i = e / nb, q = e % nb;
            const uint16_t k = __ldg((const uint16_t*)src.kd + (sa + s.src[i]) * nb + q), v = __ldg((const uint16_t*)src.vd + (sa + s.src[i]) * nb + q);
            ((uint16_t*)dst.kd)[(da + w0) * nb + e] = k;
            ((uint16_t*)dst.vd)[(da + w0) * nb + e] = v;
        }
        for (int i = tid; i < rows; i += ET) {
            if (mass_out) mass_out[(size_t)head * dst.cap + w0 + i] = m[s.src[i]];
            if (kept) kept[(size_t)head * budget + w0 + i] = s.src[i];
        }
    }
}

}  // namespace

int launch_kv4_append(const Kv4& c, const float* k, const float* v, int ldkv, const KvRows& rows, int max_rows, const int* lens, cudaStream_t st) {
    const long long warps = (long long)max_rows << (c.nb > 4);
    const dim3 grid((unsigned)std::min<long long>((warps + 7) / 8, 4096), c.n_kv, c.n_seq);
    FC_CUDA(launch_pdl(kv4_append_kernel, grid, dim3(256), 0, st, c, k, v, ldkv, rows, lens));
    FC_LAUNCHED();
    return FC_OK;
}

int kv4_make(Arena& arena, int n_seq, int n_kv, int dim, int cap, Kv4* c) {
    const int pad = (cap + kKvTile - 1) / kKvTile * kKvTile;
    const size_t rows = (size_t)n_seq * n_kv * pad, q = rows * dim / 2, d = rows * (dim / kKvBlock) * 2;
    // one allocation: rows are padded to 64, so that each part is a multiple of 128 bytes
    char* p = nullptr;
    FC_TRY(arena.alloc((void**)&p, 2 * (q + d)));
    FC_CUDA(cudaMemset(p, 0, 2 * (q + d)));
    FC_CUDA(cudaStreamSynchronize(0));
    *c = Kv4{(uint32_t*)p, (uint32_t*)(p + q), (__half*)(p + 2 * q), (__half*)(p + 2 * q + d), n_seq, n_kv, dim / kKvBlock, cap, pad};
    return FC_OK;
}

int launch_kv4_evict(const Kv4& a, const Kv4& b, const int* lens, int* lens_out, int budget, int recent, const float* mass, float* mass_out, int* kept, int device,
                     cudaStream_t st, const StepState* state) {
    static bool attr_set[64] = {};
    if (device >= 64 || !attr_set[device]) {
        FC_CUDA(cudaFuncSetAttribute(kv4_evict_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(EvictShared)));
        if (device < 64) attr_set[device] = true;
    }
    // CTAs that share a head: one an SM, as each looks for the cut (512 threads and two an SM: 33.3 us for 64 heads of 16001, so 26.9); 64
    // rows of dst each at least
    const long long heads = (long long)a.n_kv * a.n_seq;
    int share = 1;
    while (share < 32 && heads * share * 2 <= 148 && budget >= share * 2 * 64) share *= 2;
    FC_CUDA(launch_pdl(kv4_evict_kernel, dim3(share, a.n_kv, a.n_seq), dim3(ET), sizeof(EvictShared), st, a, b, lens, lens_out, budget, recent, mass, mass_out, kept, state));
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
    const int rc = kv4_make(c->arena, n_seq, n_kv_head, head_dim, capacity, &c->c);
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
    if (!aligned16(k) || !aligned16(v)) return fail(FC_E_ARG, "fc_kv4_read_dev: k and v must be 16-byte aligned");
    const int per = 128 / (c->c.nb * 4);
    const dim3 grid((unsigned)std::min<long long>(((long long)n * c->c.n_kv + per - 1) / per, std::max(1, 148 * 16 / c->c.n_seq)), c->c.n_seq);
    FC_CUDA(launch_pdl(kv4_read_kernel, grid, dim3(256), 0, (cudaStream_t)stream, c->c, from, n, k, v));
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
    return launch_kv4_evict(a, b, lens, lens_out, budget, recent, mass, mass_out, kept, src->device, (cudaStream_t)stream);
}

}  // extern "C"
