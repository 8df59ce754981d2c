// Draws from rows of logits on the device with given random numbers: temperature -> top-k -> top-p -> min-p -> the first id at which
// the running mass of what stays reaches u times its whole. The filters are those of sample.cu (all of a tie at a cut stays), and each of them
// keeps what lies above a value of its own: top-k the k-th largest logit, top-p the largest logit down to which the mass reaches
// top_p of the whole row, min-p the logit whose weight is min_p of the largest. They therefore commute, and the row is never sorted.
//
// Weights are exp((l - max) / T), computed in f64 and summed as whole numbers of 2^-42: a flat row of 2^17 ids has borders 2^-17 apart, of
// which sums in 32 bits miss one in a hundred; whole numbers can be added in any order (each is off by half of 2^-42 of the largest at most). The exponential is Tang's (Table-driven
// implementation of the exponential function, ACM TOMS 15, 1989): 2^(i / 64) from a table, times a polynomial of degree 3, to 4e-11.
//
// A cluster of CTAs shares a row and passes over it two or three times: (1) the largest and the least; (2) for a top-k or top-p, counts
// and f32 masses by value in 2048 buckets, which say in which few of them the cut lies; (3) the exact weights, summed
// by chunk above those buckets, listed in them. The list gives the cut, exactly; if it does not hold the cut after all, or not all of
// them, bisection finds it. The chunk that the random number falls into is walked by one warp.
//
// Bound: the instructions of the passes (a weight is 10 operations in f64 and some forty in all), and for few rows their latency. 192 rows of
// 131072: 25 us for the largest, 80 for a draw without filters, 186 with top-p 0.98, 148 with it in every other row; a row of 32000 with all filters 19 us.
#include <cooperative_groups.h>

#include <cfloat>

#include "pdl.cuh"

namespace fc {

namespace {

namespace cg = cooperative_groups;

constexpr int RT = 256, RW = RT / 32, BUCKETS = 2048, PER = BUCKETS / RT, LIST = 1024, CHUNKS = 512;
constexpr int kFix = 42;                      // weights are whole numbers of 2^-42; rows of up to 2^20 of them stay below 2^63
constexpr int kMaxVocab = 1 << 20;
constexpr int kPairs = 160;                   // entries of a list that are compared each with each (at most a thread each)
constexpr int kSlice = 40960;                 // ids of a CTA that shared memory holds
constexpr double kLeast = -40.0;              // weights under 2^-40 are not drawn
using u64 = unsigned long long;

// Logits in their order as unsigned keys, and back.
__device__ __forceinline__ unsigned logit_key(float l) {
    const unsigned b = __float_as_uint(l + 0.0f);
    return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float key_logit(unsigned k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }

struct Row {
    const float* p;
    int V;
    bool vec;                                 // 16-byte aligned
    // NaN is a forbidden id, as -inf
    static __device__ __forceinline__ float fix(float l) { return fmaxf(l, -INFINITY); }
    // four ids from i on as they are: a load in flight has no reader yet
    __device__ __forceinline__ float4 load4(int i) const {
        if (vec && i + 3 < V) return __ldg((const float4*)(p + i));
        float4 v;
        v.x = i < V ? __ldg(p + i) : -INFINITY;
        v.y = i + 1 < V ? __ldg(p + i + 1) : -INFINITY;
        v.z = i + 2 < V ? __ldg(p + i + 2) : -INFINITY;
        v.w = i + 3 < V ? __ldg(p + i + 3) : -INFINITY;
        return v;
    }
};

struct Weigher {
    double scale, largest;                    // log2(e) / T
    float least;                              // logits below it weigh nothing (2^-45 at most): they are not asked for
    float top;                                // asked for in the place of what does not count
    const double* table;
    // the difference first (of two f32 it is next to exact): the largest is 0 whatever its size, where a rounded product of it would leave its rounding
    __device__ __forceinline__ double log2w(float l) const { return ((double)l - largest) * scale; }
    // 2^(x + up) - z, z its table entry with the exponent, for -1000 <= x <= 0: x = (64 n + i) / 64 + r, |r| <= 1 / 128
    __device__ __forceinline__ double power(double x, int up, double* z) const {
        const double magic = 6755399441055744.0 / 64.0;      // 1.5 * 2^52 / 64: the sum's last bits are 64 x, rounded
        const double t = x + magic;
        const int k = __double2loint(t);
        const double r = x - (t - magic), e = table[k & 63];
        *z = __hiloint2double(__double2hiint(e) + ((k >> 6) + up) * (1 << 20), __double2loint(e));
        return r * fma(r, fma(r, 5.5504108664821580e-2, 2.4022650695910071e-1), 6.9314718055994531e-1);
    }
    // the sum's last bits are the weight in units of 2^-42, rounded; 0 for what does not count
    __device__ __forceinline__ u64 fixed(float l, bool counts = true) const {
        double z;
        const double q = power(log2w(counts ? l : top), kFix, &z);
        z = __hiloint2double(counts ? __double2hiint(z) : 0, __double2loint(z));
        return (u64)__double_as_longlong(fma(z, q, z + 4503599627370496.0)) & 0xfffffffffffffull;
    }
    __device__ __forceinline__ double exact(float l) const {
        double z;
        const double q = power(log2w(l), 0, &z);
        return fma(z, q, z);
    }
};

__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

struct __align__(16) Shared {
    unsigned cnt[BUCKETS], mass[BUCKETS];                 // this CTA's buckets
    union {
        struct {                                          // the cluster's, until the cut's buckets are known
            unsigned all_cnt[BUCKETS];
            float all_mass[BUCKETS];
        };
        struct {                                          // what lies in them
            u64 list_w[LIST];
            unsigned list_key[LIST];
            unsigned short list_chunk[LIST];
        };
    };
    u64 chunk[CHUNKS];
    double table[64];
    u64 warp_w[RW], above_w, list_all, whole, sum;
    float warp_f[RW];
    unsigned warp_n[RW];
    float most, least, tops[RW], lows[RW];
    int first, firsts[RW];
    int listed, b1, b2;
    unsigned above_n, cut, found;
    unsigned pair_n[2][RW];
    u64 pair_w[2][RW];
    u64 wide_w;                                           // sums of a pass of the bisection
    unsigned wide_n;
};

static_assert(sizeof(Shared) % 16 == 0, "the slice behind it is read in 16-byte words");

// The ids that a CTA holds, in chunks that the warps take in turn: in shared memory (slice) behind the first pass where they fit.
struct Share {
    Row row;
    int begin, end, chunk;
    float* slice;
    bool endless;                             // the largest is infinite: among infinities the others weigh nothing
    __device__ __forceinline__ float settle(float l) const { return endless ? (l == INFINITY ? 0.0f : -INFINITY) : l; }
    __device__ __forceinline__ float at(int i) const { return settle(slice ? slice[i - begin] : Row::fix(__ldg(row.p + i))); }
    // f(values, chunk) for four ids a lane, f.done(chunk) behind each chunk; up to four loads of a lane are on their way
    template <class F>
    __device__ __forceinline__ void over(const F& f) const {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, steps = chunk / 128;
        auto give = [&](const float4& x, int c) {
            float v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = Row::fix(v[e]);
            if (endless) {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = settle(v[e]);
            }
            f(v, c);
        };
        const float4 none = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        if (slice) {
            for (int c = warp, i0 = begin + warp * chunk; i0 < end; c += RW, i0 += RW * chunk) {
                for (int q = 0; q < steps; ++q)
                    if (i0 + 128 * q < end) give(*(const float4*)(slice + i0 - begin + 128 * q + 4 * lane), c);
                f.done(c);
            }
            return;
        }
        // the warp's pieces of 128 ids in order: piece j is step j % steps (a power of two) of its chunk j / steps
        const int bits = 31 - __clz(steps);
        const int chunks = end > begin + warp * chunk ? (end - begin - warp * chunk + RW * chunk - 1) / (RW * chunk) : 0, pieces = chunks * steps;
        auto place = [&](int j) { return begin + (warp + (j >> bits) * RW) * chunk + (j & (steps - 1)) * 128 + 4 * lane; };
        for (int j0 = 0; j0 < pieces; j0 += 4) {
            float4 x[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int i = place(j0 + q);
                x[q] = j0 + q < pieces && i < end ? row.load4(i) : none;
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int j = j0 + q;
                if (j >= pieces) break;
                const int c = warp + (j >> bits) * RW;
                give(x[q], c);
                if (((j + 1) & (steps - 1)) == 0) f.done(c);
            }
        }
    }
};

// The i-th row, of each RT rows those with top-k or top-p first (two passes more), then draws without, then the first of the largest. All
// threads; count: RW + 1 words, free again behind the call.
__device__ __forceinline__ int row_by_work(const fc_row_sampling* __restrict__ params, int n_rows, int V, int i, int* count) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, base = i - i % RT;
    int work = -1;
    if (base + tid < n_rows) {
        const fc_row_sampling p = params[base + tid];
        work = !(p.temperature > 0.0f) ? 0 : (p.top_k > 0 && p.top_k < V) || p.top_p < 1.0f ? 2 : 1;
    }
    const unsigned much = __ballot_sync(0xffffffffu, work == 2), some = __ballot_sync(0xffffffffu, work == 1), little = __ballot_sync(0xffffffffu, work == 0);
    if (lane == 0) count[warp] = __popc(much) | __popc(some) << 10 | __popc(little) << 20;
    __syncthreads();
    int before = 0, all = 0;
    for (int w = 0; w < RW; ++w) {
        if (w < warp) before += count[w];
        all += count[w];
    }
    const unsigned ahead = (1u << lane) - 1;
    const int n2 = all & 1023, n1 = all >> 10 & 1023;
    const int place = work == 2 ? (before & 1023) + __popc(much & ahead)
                    : work == 1 ? n2 + (before >> 10 & 1023) + __popc(some & ahead) : n2 + n1 + (before >> 20) + __popc(little & ahead);
    if (work >= 0 && place == i - base) count[RW] = base + tid;
    __syncthreads();
    const int row = count[RW];
    __syncthreads();
    return row;
}

__global__ void __launch_bounds__(RT, 4) sample_rows_kernel(const float* __restrict__ logits, long long ld, int V, const fc_row_sampling* __restrict__ params,
                                                            const float* __restrict__ u, int* __restrict__ token, float* __restrict__ prob, int cs, int chunk, int in_shared, int n_rows, int by_work) {
    extern __shared__ __align__(16) char smem_raw[];
    Shared& s = *(Shared*)smem_raw;
    cg::cluster_group cluster = cg::this_cluster();
    pdl_wait();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rank = blockIdx.x % cs;
    const int r = by_work ? row_by_work(params, n_rows, V, blockIdx.x / cs, (int*)smem_raw) : blockIdx.x / cs;
    const fc_row_sampling p = params[r];
    const float* const in = logits + (size_t)r * ld;
    // whole chunks a CTA
    const int share = ((V + cs - 1) / cs + chunk - 1) / chunk * chunk, begin = min(V, rank * share), end = min(V, begin + share);
    Share ids = {{in, V, ((uintptr_t)in & 15) == 0}, begin, end, chunk, in_shared ? (float*)(smem_raw + sizeof(Shared)) : nullptr, false};
    auto sync = [&]() { if (cs > 1) cluster.sync(); else __syncthreads(); };
    auto at = [&](auto* x, int q) { return cs > 1 ? cluster.map_shared_rank(x, q) : x; };

    // 1. the largest, where it comes first, and the least finite one; four loads of a lane on their way at a time
    float top = -INFINITY, low = INFINITY;
    int first = V;
    for (int i0 = begin; i0 < end; i0 += 16 * RT) {
        float4 x[4];
        if (ids.row.vec && i0 + 16 * RT <= end) {
#pragma unroll
            for (int q = 0; q < 4; ++q) x[q] = __ldg((const float4*)(in + i0 + 4 * (q * RT + tid)));
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q) x[q] = ids.row.load4(i0 + 4 * (q * RT + tid));
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int i = i0 + 4 * (q * RT + tid);
            if (i >= end) continue;
            const float v[4] = {Row::fix(x[q].x), Row::fix(x[q].y), Row::fix(x[q].z), Row::fix(x[q].w)};
            if (ids.slice) *(float4*)(ids.slice + i - begin) = make_float4(v[0], v[1], v[2], v[3]);
            const float most = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
            if (most > top) {
                top = most;
                first = i + (v[0] == most ? 0 : v[1] == most ? 1 : v[2] == most ? 2 : 3);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) low = fminf(low, v[e] > -INFINITY ? v[e] : INFINITY);
        }
    }
    // what a chunk's last quarters read behind the end
    if (ids.slice)
        for (int i = ((end - begin + 3) & ~3) + tid; i < share; i += RT) ids.slice[i] = -INFINITY;
    if (tid < 64) s.table[tid] = exp2((double)tid * 0.015625);
    for (int b = tid; b < BUCKETS; b += RT) s.cnt[b] = s.mass[b] = 0;
    auto better = [](float a, int i, float b, int j) { return a > b || (a == b && i < j); };
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float t2 = __shfl_xor_sync(0xffffffffu, top, o), l2 = __shfl_xor_sync(0xffffffffu, low, o);
        const int f2 = __shfl_xor_sync(0xffffffffu, first, o);
        if (better(t2, f2, top, first)) { top = t2; first = f2; }
        low = fminf(low, l2);
    }
    if (lane == 0) { s.tops[warp] = top; s.lows[warp] = low; s.firsts[warp] = first; }
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < RW; ++w) {
            if (better(s.tops[w], s.firsts[w], top, first)) { top = s.tops[w]; first = s.firsts[w]; }
            low = fminf(low, s.lows[w]);
        }
        s.most = top; s.least = low; s.first = first;
        s.listed = 0; s.b1 = s.b2 = BUCKETS; s.found = 0;
    }
    sync();
    top = -INFINITY; low = INFINITY; first = V;
    for (int q = 0; q < cs; ++q) {
        const float t2 = *at(&s.most, q);
        const int f2 = *at(&s.first, q);
        if (better(t2, f2, top, first)) { top = t2; first = f2; }
        low = fminf(low, *at(&s.least, q));
    }
    if (top == -INFINITY || !(p.temperature > 0.0f)) {
        // nothing can be drawn, or the first of the largest
        if (rank == 0 && tid == 0) { token[r] = top == -INFINITY ? -1 : first; if (prob) prob[r] = top == -INFINITY ? 0.0f : 1.0f; }
        if (cs > 1) cluster.sync();           // no rank leaves while another reads its memory
        return;
    }
    ids.endless = top == INFINITY;
    if (ids.endless) { top = low = 0.0f; }

    const double temp = fmin(fmax((double)p.temperature, 0.01), 1e30);
    // (45 / log2(e) = 31.2; a rounding of the difference or the product does not reach 2^-43)
    const double scale = 1.4426950408889634 / temp;
    const Weigher weigh = {scale, (double)top, fmaxf(top - 31.25f * (float)temp, -FLT_MAX), top, s.table};
    const bool cut_k = p.top_k > 0 && p.top_k < V, cut_p = p.top_p < 1.0f;
    // the least logit that min-p, and 2^-40, let stay: the weight falls with the logit, so that one comparison in f32 decides
    const double floor_x = p.min_p > 0.0f ? fmax(log2(fmin((double)p.min_p, 1.0)), kLeast) : kLeast;
    // (never above the largest, which always stays, nor below what is finite: -inf weighs nothing)
    float keep = (float)fmax((double)top + floor_x / scale, -(double)FLT_MAX);
    for (int i = 0; i < 4 && keep > -FLT_MAX && weigh.log2w(keep) >= floor_x; ++i) keep = nextafterf(keep, -INFINITY);
    for (int i = 0; i < 8 && keep < top && weigh.log2w(keep) < floor_x; ++i) keep = nextafterf(keep, INFINITY);

    u64 lane_sum = 0, warp_all = 0, lane_all = 0;
    // the weights of what is not below `keep`, by chunk; a chunk's lanes without any skip them
    struct Keep {
        Shared& s;
        const Weigher& weigh;
        float keep;
        int lane;
        u64& sum;
        u64& all;
        __device__ __forceinline__ void operator()(const float (&v)[4], int) const {
            if (!__any_sync(0xffffffffu, fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])) >= keep)) return;
#pragma unroll
            for (int e = 0; e < 4; ++e) sum += weigh.fixed(v[e], v[e] >= keep);
        }
        __device__ __forceinline__ void done(int c) const {
            const u64 w = warp_sum(sum);
            all += w;
            sum = 0;
            if (lane == 0) s.chunk[c] = w;
        }
    };
    if (!cut_k && !cut_p) {
        ids.over(Keep{s, weigh, keep, lane, lane_sum, warp_all});
    } else {
        // 2. buckets of even width from the largest down to what has a weight. A bucket's mass is in units of a
        // part of its middle's weight, as small as all ids in one bucket allow.
        const float range = fminf(top - low, 31.25f * (float)temp), per = range > 0.0f ? (float)(BUCKETS - 1) / range : 0.0f;
        const float unit = (float)(1u << min(30 - (32 - __clz(V)), 22)), slope = (float)weigh.scale, width = range > 0.0f ? range / (float)(BUCKETS - 1) * slope : 0.0f;      // in powers of two
        // (2^23 + n has n in its low bits)
        auto bucket_of = [&](float l) { return __float_as_int(fminf((top - l) * per, (float)(BUCKETS - 1)) + 8388608.0f) & (2 * BUCKETS - 1); };
        struct Sort {
            Shared& s;
            const decltype(bucket_of)& bucket;
            float top, slope, width, unit;
            bool count_too, mass_too;
            __device__ __forceinline__ void operator()(const float (&v)[4], int) const {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int b = bucket(v[e]);
                    if (count_too && v[e] > -INFINITY) atomicAdd(&s.cnt[b], 1u);
                    if (mass_too) {
                        // (in the last bucket, what lies behind the range comes to nothing)
                        const float x = fmaf(v[e] - top, slope, (float)b * width);
                        float w;
                        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w) : "f"(x));
                        const unsigned m = (unsigned)__float_as_int(fmaf(w, unit, 8388608.0f)) - 0x4b000000u;
                        if (m) atomicAdd(&s.mass[b], m);
                    }
                }
            }
            __device__ __forceinline__ void done(int) const {}
        };
        ids.over(Sort{s, bucket_of, top, slope, width, unit, cut_k, cut_p});
        sync();
        // each rank adds up its share of the buckets and hands it to all
        for (int b = rank * RT + tid; b < BUCKETS; b += cs * RT) {
            unsigned n = 0;
            u64 m = 0;
            for (int q = 0; q < cs; ++q) {
                n += *at(&s.cnt[b], q);
                m += *at(&s.mass[b], q);
            }
            const float mass = (float)m * exp2f(-(float)b * width);
            for (int q = 0; q < cs; ++q) { *at(&s.all_cnt[b], q) = n; *at(&s.all_mass[b], q) = mass; }
        }
        sync();
        // PER buckets a thread: how many ids and how much mass there are at the end of each
        unsigned bn[PER], n = 0;
        float bm[PER], m = 0.0f;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            n += s.all_cnt[PER * tid + i]; bn[i] = n;
            m += s.all_mass[PER * tid + i]; bm[i] = m;
        }
        unsigned an = n;
        float am = m;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned n2 = __shfl_up_sync(0xffffffffu, an, o);
            const float m2 = __shfl_up_sync(0xffffffffu, am, o);
            if (lane >= o) { an += n2; am += m2; }
        }
        if (lane == 31) { s.warp_n[warp] = an; s.warp_f[warp] = am; }
        __syncthreads();
        float all_m = 0.0f;
        for (int q = 0; q < RW; ++q) {
            if (q < warp) { an += s.warp_n[q]; am += s.warp_f[q]; }
            all_m += s.warp_f[q];
        }
        an -= n; am -= m;
        // the cut lies behind b1 - 1 and not behind b2: ids are counted, the mass is sure to half a unit of weights of 0.98 units and above, and
        // to the roundings in f32 of a logarithm below 2^6
        const float want_m = p.top_p * all_m, slack = all_m * (0.6f / unit + 1.5e-5f);
        int b1 = BUCKETS, b2 = BUCKETS;
#pragma unroll
        for (int i = PER - 1; i >= 0; --i) {
            const bool k = cut_k && an + bn[i] >= (unsigned)p.top_k;
            if (k || (cut_p && am + bm[i] >= want_m - slack)) b1 = PER * tid + i;
            if (k || (cut_p && am + bm[i] >= want_m + slack)) b2 = PER * tid + i;
        }
        if (b1 < BUCKETS) atomicMin(&s.b1, b1);
        if (b2 < BUCKETS) atomicMin(&s.b2, b2);
        __syncthreads();
        b1 = s.b1; b2 = min(s.b2, BUCKETS - 1);
        sync();                               // the list lies where the buckets were
        if (b1 - 1 >= PER * tid && b1 - 1 < PER * (tid + 1)) s.above_n = an + bn[(b1 - 1) % PER];
        if (b1 == 0 && tid == 0) s.above_n = 0;

        // 3. the weights: above those buckets by chunk, in them listed, below them only for the whole
        struct List {
            Shared& s;
            const Weigher& weigh;
            const decltype(bucket_of)& bucket;
            float keep;
            int b1, b2, lane;
            bool whole;
            u64& sum;
            u64& all;
            u64& above;
            __device__ __forceinline__ void operator()(const float (&v)[4], int c) const {
                const float most = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
                if (!__any_sync(0xffffffffu, (whole ? most >= weigh.least : most > -INFINITY && bucket(most) <= b2))) return;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const u64 w = weigh.fixed(v[e], v[e] >= weigh.least);
                    const int b = bucket(v[e]);
                    all += w;
                    above += b < b1 ? w : 0;
                    sum += b < b1 && v[e] >= keep ? w : 0;
                    if (b >= b1 && b <= b2 && v[e] > -INFINITY) {
                        const int q = atomicAdd(&s.listed, 1);
                        if (q < LIST) { s.list_key[q] = logit_key(v[e]); s.list_w[q] = w; s.list_chunk[q] = (unsigned short)c; }
                    }
                }
            }
            __device__ __forceinline__ void done(int c) const {
                const u64 w = warp_sum(sum);
                sum = 0;
                if (lane == 0) s.chunk[c] = w;
            }
        };
        u64 lane_above = 0;
        ids.over(List{s, weigh, bucket_of, keep, b1, b2, lane, cut_p, lane_sum, lane_all, lane_above});
        lane_all = warp_sum(lane_all);
        lane_above = warp_sum(lane_above);
        __syncthreads();                      // the warps' sums of the buckets have been read
        if (lane == 0) { s.warp_w[warp] = lane_all; s.list_all = 0; s.above_w = 0; }
        __syncthreads();
        if (lane == 0) atomicAdd(&s.above_w, lane_above);
        if (tid == 0) {
            u64 w = 0;
            for (int q = 0; q < RW; ++q) w += s.warp_w[q];
            s.whole = w;
        }
        sync();
        u64 whole = 0, above_w = 0;
        int total = 0;
        for (int q = 0; q < cs; ++q) { whole += *at(&s.whole, q); above_w += *at(&s.above_w, q); total += *at(&s.listed, q); }
        const unsigned above_n = s.above_n;
        const double want = (double)p.top_p * (double)whole;
        auto enough = [&](unsigned k, u64 w) { return (cut_k && k >= (unsigned)p.top_k) || (cut_p && (double)w >= want); };
        unsigned cut = 0;
        // no id, or not enough mass even at the end: nothing is cut
        const bool some = b1 < BUCKETS;
        bool sure = !some || (total <= LIST && !(b1 > 0 && enough(above_n, above_w)));
        if (some && sure) {
            if (rank == 0) {
                // rank 0 gathers the list behind its own, and looks for the largest key down to which k ids, or the mass, are there
                for (int q = 1, base = s.listed; q < cs; ++q) {
                    const int other = *at(&s.listed, q);
                    const unsigned* keys = at(s.list_key, q);
                    const u64* ws = at(s.list_w, q);
                    for (int i = tid; i < other; i += RT) { s.list_key[base + i] = keys[i]; s.list_w[base + i] = ws[i]; }
                    base += other;
                }
                __syncthreads();
                if (total <= kPairs) {
                    // each with each; all of a tie write the same
                    const unsigned key = tid < total ? s.list_key[tid] : 0;
                    unsigned ge = above_n, gt = above_n;
                    u64 wge = above_w, wgt = above_w;
                    for (int j = 0; j < total; ++j) {
                        const unsigned k = s.list_key[j];
                        const u64 x = s.list_w[j];
                        if (k >= key) { ++ge; wge += x; }
                        if (k > key) { ++gt; wgt += x; }
                    }
                    if (tid < total && enough(ge, wge) && (gt == 0 || !enough(gt, wgt)))
                        for (int q = 0; q < cs; ++q) { *at(&s.cut, q) = key; *at(&s.found, q) = 1; }
                } else {
                    // by the bits in which they differ
                    constexpr int EACH = LIST / RT;
                    unsigned key[EACH], most = 0, least = 0xffffffffu;
                    u64 x[EACH];
#pragma unroll
                    for (int e = 0; e < EACH; ++e) {
                        const int i = tid + e * RT;
                        key[e] = i < total ? s.list_key[i] : 0;
                        x[e] = i < total ? s.list_w[i] : 0;
                        most = max(most, key[e]);
                        least = min(least, i < total ? key[e] : 0xffffffffu);
                    }
                    most = __reduce_max_sync(0xffffffffu, most);
                    least = __reduce_min_sync(0xffffffffu, least);
                    if (lane == 0) { s.warp_n[warp] = most; s.pair_n[0][warp] = least; }
                    __syncthreads();
                    for (int q = 0; q < RW; ++q) { most = max(most, s.warp_n[q]); least = min(least, s.pair_n[0][q]); }
                    __syncthreads();
                    const int bits = 32 - __clz(most ^ least);
                    unsigned c = bits < 32 ? most >> bits << bits : 0;
                    bool reached = false;
                    for (int bit = bits; bit >= 0; --bit) {           // (first what they have in common)
                        const unsigned cand = bit == bits ? c : c | 1u << bit;
                        unsigned n = 0;
                        u64 w = 0;
#pragma unroll
                        for (int e = 0; e < EACH; ++e)
                            if (key[e] >= cand && tid + e * RT < total) { ++n; w += x[e]; }
                        n = __reduce_add_sync(0xffffffffu, n);
                        w = warp_sum(w);
                        if (lane == 0) { s.pair_n[bit & 1][warp] = n; s.pair_w[bit & 1][warp] = w; }
                        __syncthreads();
                        n = above_n; w = above_w;
                        for (int q = 0; q < RW; ++q) { n += s.pair_n[bit & 1][q]; w += s.pair_w[bit & 1][q]; }
                        if (n && enough(n, w)) { c = cand; reached = true; }      // (n: a top-p of 0 is reached ahead of the first id)
                    }
                    if (tid == 0 && reached)
                        for (int q = 0; q < cs; ++q) { *at(&s.cut, q) = c; *at(&s.found, q) = 1; }
                }
            }
            sync();
            sure = s.found != 0;
            // not in the list though the buckets end behind it: the mass is never reached, and nothing is cut
            if (!sure && s.b2 == BUCKETS) sure = true;
            else cut = sure ? s.cut : 0;
        }
        if (!sure) {
            // the cut's bits from the highest down, a pass each over what is not above those buckets
            struct Count {
                const Weigher& weigh;
                const decltype(bucket_of)& bucket;
                int from;
                unsigned cand;
                bool mass_too;
                unsigned& n;
                u64& w;
                __device__ __forceinline__ void operator()(const float (&v)[4], int) const {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (v[e] > -INFINITY && logit_key(v[e]) >= cand && bucket(v[e]) >= from) {
                            ++n;
                            if (mass_too && v[e] >= weigh.least) w += weigh.fixed(v[e]);
                        }
                }
                __device__ __forceinline__ void done(int) const {}
            };
            const bool before = b1 > 0 && enough(above_n, above_w);       // (the f32 masses were wrong: from the start)
            cut = 0;
            for (int bit = 31; bit >= 0; --bit) {
                const unsigned cand = cut | (1u << bit);
                unsigned n = 0;
                u64 w = 0;
                ids.over(Count{weigh, bucket_of, before ? 0 : b1, cand, cut_p, n, w});
                n = __reduce_add_sync(0xffffffffu, n);
                w = warp_sum(w);
                __syncthreads();
                if (lane == 0) { s.warp_n[warp] = n; s.warp_w[warp] = w; }
                __syncthreads();
                if (tid == 0) {
                    for (int q = 1; q < RW; ++q) { n += s.warp_n[q]; w += s.warp_w[q]; }
                    s.wide_n = n; s.wide_w = w;
                }
                sync();
                n = 0; w = 0;
                for (int q = 0; q < cs; ++q) { n += *at(&s.wide_n, q); w += *at(&s.wide_w, q); }
                if (n && enough(before ? n : above_n + n, before ? w : above_w + w)) cut = cand;
                sync();
            }
            if (cut) keep = fmaxf(keep, key_logit(cut));
            ids.over(Keep{s, weigh, keep, lane, lane_sum, warp_all});
        } else {
            if (cut) keep = fmaxf(keep, key_logit(cut));
            // what stays of the list joins its chunks
            __syncthreads();
            const int mine = min(s.listed, LIST);
            for (int i = tid; i < mine; i += RT)
                if (key_logit(s.list_key[i]) >= keep) atomicAdd(&s.chunk[s.list_chunk[i]], s.list_w[i]);
            __syncthreads();
            const int chunks = (end - begin + chunk - 1) / chunk;
            for (int i = tid; i < chunks; i += RT) lane_sum += s.chunk[i];
            warp_all = warp_sum(lane_sum);
        }
        __syncthreads();                      // the warps' sums of the pass have been read
    }
    // (earlier, the next draw's CTAs would take their places among this one's: 192 rows of 131072 in 199 us, so 174)
    pdl_trigger();
    if (lane == 0) s.warp_w[warp] = warp_all;
    __syncthreads();
    if (tid == 0) {
        u64 w = 0;
        for (int q = 0; q < RW; ++q) w += s.warp_w[q];
        s.sum = w;
    }
    sync();
    u64 whole = 0, before = 0;
    for (int q = 0; q < cs; ++q) {
        const u64 w = *at(&s.sum, q);
        if (q < rank) before += w;
        whole += w;
    }
    const double aim = fmin(fmax((double)u[r], 0.0), 1.0) * (double)whole;
    const u64 mine = s.sum;
    // the running mass reaches u times the whole where it first is at least that; the largest id always has mass
    auto there = [&](u64 m) { return m > 0 && (double)m >= aim; };
    if (there(before + mine) && !there(before) && warp == 0) {
        // one warp of one rank: the chunk, then the id
        const int n = (end - begin + chunk - 1) / chunk;
        u64 run = before;
        int c0 = 0;
        for (;; c0 += 32) {
            const u64 w = c0 + lane < n ? s.chunk[c0 + lane] : 0;
            u64 incl = w;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const u64 x = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += x;
            }
            const unsigned hit = __ballot_sync(0xffffffffu, there(run + incl));
            if (hit || c0 + 32 >= n) {
                const int q = hit ? __ffs(hit) - 1 : 31;
                run += __shfl_sync(0xffffffffu, incl - w, q);
                c0 += q;
                break;
            }
            run += __shfl_sync(0xffffffffu, incl, 31);
        }
        const int per_lane = chunk / 32, i0 = begin + c0 * chunk + lane * per_lane, i1 = min(i0 + per_lane, end);
        auto weight = [&](int i) -> u64 {
            const float l = ids.at(i);
            return l >= keep ? weigh.fixed(l) : 0;
        };
        u64 w = 0;
        for (int i = i0; i < i1; ++i) w += weight(i);
        u64 incl = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 x = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += x;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, there(run + incl));
        if (hit && lane == __ffs(hit) - 1) {
            u64 m = run + incl - w;
            int i = i0;
            for (; i < i1; ++i) {
                m += weight(i);
                if (there(m)) break;
            }
            token[r] = i;
            if (prob) prob[r] = (float)(weigh.exact(ids.at(i)) * (double)(1ull << kFix) / (double)whole);
        }
    }
    if (cs > 1) cluster.sync();               // no rank leaves while another reads its memory
}

}  // namespace
}  // namespace fc

using namespace fc;

extern "C" int fc_sample_rows_dev(int device, const float* logits, int64_t ld, int n_rows, int vocab, const fc_row_sampling* params, const float* u,
                                  int32_t* token, float* prob, void* stream) {
    if (!logits || !params || !u || !token) return fail(FC_E_ARG, "fc_sample_rows_dev: null argument");
    if (n_rows < 0 || vocab <= 0 || vocab > kMaxVocab || ld < vocab)
        return fail(FC_E_SHAPE, "fc_sample_rows_dev: %d rows of %d logits (1..%d), %lld apart", n_rows, vocab, kMaxVocab, (long long)ld);
    if (!aligned16(params)) return fail(FC_E_ARG, "fc_sample_rows_dev: params must be 16-byte aligned");
    if (!n_rows) return FC_OK;
    static bool ready[64] = {};
    static int resident[64][2][9];                // clusters of so many CTAs, with a slice in shared memory or without, that the device holds at once
    int here[2][9], (*const room)[9] = device >= 0 && device < 64 ? resident[device] : here;
    constexpr int kSmall = kSlice / 8;            // ids that CTAs which share an SM may hold in shared memory
    if (device < 0 || device >= 64 || !ready[device]) {
        FC_TRY(select_device(device));
        FC_CUDA(cudaFuncSetAttribute(sample_rows_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(Shared) + kSlice * sizeof(float)));
        for (int cs = 1; cs <= 8; ++cs)
            for (int in = 0; in < 2; ++in)
                FC_CUDA(resident_clusters((const void*)sample_rows_kernel, dim3(RT), sizeof(Shared) + in * kSmall * sizeof(float), cs, &room[in][cs]));
        if (device < 64) ready[device] = true;
    } else {
        int current = -1;
        FC_CUDA(cudaGetDevice(&current));
        if (current != device) FC_CUDA(cudaSetDevice(device));
    }
    // a CTA costs some microseconds whatever it holds: no more of them than are resident, 1024 ids each at least (128 rows of 131072, top-p: 4
    // CTAs a row 126 us, 2 148; 192 rows: 2 CTAs 187 us, 3, of which not all are resident, 210)
    int cs = 1, chunk = 128;
    for (int x = 2; x <= 8; ++x)
        if (n_rows <= room[vocab <= kSmall * x][x] && x * 1024 <= vocab) cs = x;
    while ((vocab + cs - 1) / cs > chunk * (CHUNKS - 1)) chunk *= 2;
    const int share = ((vocab + cs - 1) / cs + chunk - 1) / chunk * chunk;
    const bool in_shared = share <= kSlice && (share <= kSmall || (long long)n_rows * cs <= 148);
    // CTAs that share SMs take the rows with filters first, so that no SM has three of those and another none (192 rows of
    // 131072, half of them with top-p: 147 us, in the order of the call 171; in a uniform batch it costs a microsecond)
    const int by_work = n_rows > 1 && (long long)n_rows * cs > 148;
    FC_CUDA(launch_pdl_cluster(sample_rows_kernel, dim3((unsigned)n_rows * cs), dim3(RT), sizeof(Shared) + (in_shared ? (size_t)share * sizeof(float) : 0), cs, (cudaStream_t)stream,
                               logits, (long long)ld, vocab, params, u, token, prob, cs, chunk, (int)in_shared, n_rows, by_work));
    FC_LAUNCHED();
    return FC_OK;
}
