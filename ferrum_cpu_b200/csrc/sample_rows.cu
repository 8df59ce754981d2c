// Draws from rows of logits on the device with given random numbers: temperature -> top-k -> top-p -> min-p -> the first id at which
// the running mass of what stays reaches u times its whole. The filters are those of sample.cu (all of a tie at a cut stays), and each of them
// keeps what lies above a value of its own: top-k the k-th largest logit, top-p the largest logit down to which the mass reaches
// top_p of the whole row, min-p the logit whose weight is min_p of the largest. They therefore commute, and the row is never sorted.
//
// Weights are exp((l - max) / T), computed in f64 and summed as whole numbers of 2^-42: a flat row of 2^17 ids has borders 2^-17 apart, of
// which sums in 32 bits miss one in a hundred; whole numbers can be added in any order. The exponential is Tang's (Table-driven
// implementation of the exponential function, ACM TOMS 15, 1989): 2^(i / 16) from a table that fills the 32 banks once, times a
// polynomial of degree 5.
//
// A cluster of CTAs shares a row and reads it up to four times, from L2 after the first: (1) the largest and the least; (2) the weights,
// their sums by chunk and, if there is a top-k or top-p, by value in 1024 buckets; (3) if there is, the bucket in which the cut lies is
// listed and searched; then the chunks' sums of what stays. The chunk that the random number falls into is walked by one warp.
#include <cooperative_groups.h>

#include "fc_common.cuh"

namespace fc {

namespace {

namespace cg = cooperative_groups;

constexpr int RT = 512, RW = RT / 32, BUCKETS = 1024, LIST = 1024, CHUNKS = 512;
constexpr int kFix = 42;                      // weights are whole numbers of 2^-42; rows of up to 2^20 of them stay below 2^63
constexpr int kMaxVocab = 1 << 20;
constexpr double kLeast = -40.0;              // weights under 2^-40 are not drawn
using u64 = unsigned long long;

// Logits in their order as unsigned keys.
__device__ __forceinline__ unsigned logit_key(float l) {
    const unsigned b = __float_as_uint(l + 0.0f);
    return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}

struct Row {
    const float* p;
    int V;
    bool vec, endless;                        // 16-byte aligned; the largest is infinite
    // NaN is a forbidden id, as -inf; among infinities the others weigh nothing
    __device__ __forceinline__ float fix(float l) const {
        l = l == l ? l : -INFINITY;
        return endless ? (l == INFINITY ? 0.0f : -INFINITY) : l;
    }
    __device__ __forceinline__ void load4(int i, float (&v)[4]) const {
        if (vec && i + 3 < V) {
            const float4 x = __ldg((const float4*)(p + i));
            v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = i + e < V ? __ldg(p + i + e) : -INFINITY;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = fix(v[e]);
    }
};

struct Weigher {
    double best, scale;                       // log2(e) / T
    float least;                              // logits below it weigh nothing: 2^-45 at most
    const double* table;
    __device__ __forceinline__ double log2w(float l) const { return ((double)l - best) * scale; }
    // 2^(x + up) for -1000 <= x <= 0: x = (16 n + i) / 16 + r, |r| <= 1 / 32
    __device__ __forceinline__ double power(double x, int up) const {
        const double magic = 6755399441055744.0 / 16.0;      // 1.5 * 2^52 / 16: the sum's last bits are 16 x, rounded
        const double t = x + magic;
        const int k = __double2loint(t);
        const double r = x - (t - magic);
        double y = fma(r, 1.3333558146428443e-3, 9.6181291076284772e-3);
        y = fma(r, y, 5.5504108664821580e-2);
        y = fma(r, y, 2.4022650695910071e-1);
        y = fma(r, y, 6.9314718055994531e-1);
        y = fma(r, y, 1.0) * table[k & 15];                  // in [0.97, 2)
        return __hiloint2double(__double2hiint(y) + ((k >> 4) + up) * (1 << 20), __double2loint(y));
    }
    // the sum's last bits are the weight in units of 2^-42, rounded
    __device__ __forceinline__ u64 fixed(double x) const {
        return (u64)__double_as_longlong(power(x, kFix) + 4503599627370496.0) & 0xfffffffffffffull;
    }
    __device__ __forceinline__ double exact(double x) const { return power(x, 0); }
};

__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

struct Shared {
    unsigned cnt[BUCKETS], lo[BUCKETS], hi[BUCKETS];      // this CTA's buckets
    unsigned all_cnt[BUCKETS];                            // the cluster's
    u64 all_mass[BUCKETS];
    u64 chunk[CHUNKS];
    u64 list_w[LIST];
    unsigned list_key[LIST];
    double table[16];
    u64 warp_w[RW], whole, sum, sums[16];
    unsigned warp_n[RW];
    float most, least, tops[16], lows[16];
    int first, firsts[16];
    int listed, bucket;
    u64 above_w;
    unsigned above_n, cut;
    int wants;                                            // 1: top-k cuts in the bucket, 2: top-p does
    u64 wide_w;                                           // sums of a pass of the fallback
    unsigned wide_n;
};

// A pass over the CTA's chunks: f(values, index of the first, chunk) for four ids a lane.
template <class F>
__device__ __forceinline__ void over(const Row& row, int begin, int end, int chunk, const F& f) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int c = warp, i0 = begin + warp * chunk; i0 < end; c += RW, i0 += RW * chunk) {
        const int stop = min(i0 + chunk, end);
        for (int i = i0 + 4 * lane; i - 4 * lane < stop; i += 128) {
            float v[4];
            if (i < stop) row.load4(i, v);
            else v[0] = v[1] = v[2] = v[3] = -INFINITY;
            f(v, i, c);
        }
        f.done(c);
    }
}

__global__ void __launch_bounds__(RT, 2) sample_rows_kernel(const float* __restrict__ logits, long long ld, int V, const fc_row_sampling* __restrict__ params,
                                                            const float* __restrict__ u, int* __restrict__ token, float* __restrict__ prob, int cs, int chunk) {
    extern __shared__ __align__(16) char smem_raw[];
    Shared& s = *(Shared*)smem_raw;
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rank = blockIdx.x % cs, r = blockIdx.x / cs;
    const fc_row_sampling p = params[r];
    Row row = {logits + (size_t)r * ld, V, false, false};
    row.vec = ((uintptr_t)row.p & 15) == 0;
    // whole chunks a CTA
    const int share = ((V + cs - 1) / cs + chunk - 1) / chunk * chunk, begin = min(V, rank * share), end = min(V, begin + share);
    auto sync = [&]() { if (cs > 1) cluster.sync(); else __syncthreads(); };
    auto at = [&](auto* x, int q) { return cs > 1 ? cluster.map_shared_rank(x, q) : x; };

    // 1. the largest, where it comes first, and the least finite one
    struct Extremes {
        float &top, &low;
        int& first;
        __device__ void operator()(const float (&v)[4], int i, int) const {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (v[e] > top) { top = v[e]; first = i + e; }
                if (v[e] > -INFINITY) low = fminf(low, v[e]);
            }
        }
        __device__ void done(int) const {}
    };
    float top = -INFINITY, low = INFINITY;
    int first = V;
    over(row, begin, end, chunk, Extremes{top, low, first});
    if (tid < 16) s.table[tid] = exp2((double)tid * 0.0625);
    for (int b = tid; b < BUCKETS; b += RT) s.cnt[b] = s.lo[b] = s.hi[b] = 0;
    if (tid < CHUNKS) s.chunk[tid] = 0;
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
        s.listed = 0;
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
    row.endless = top == INFINITY;
    if (row.endless) { top = low = 0.0f; }

    const double temp = fmax((double)p.temperature, 0.01);
    // (45 / log2(e) = 31.2; a rounding of the product or the difference does not reach 2^-43)
    const Weigher weigh = {(double)top, 1.4426950408889634 / temp, top - 31.25f * (float)fmin(temp, 1e30), s.table};
    const bool cut_k = p.top_k > 0 && p.top_k < V, cut_p = p.top_p < 1.0f;
    const double floor_x = p.min_p > 0.0f ? fmax(log2(fmin((double)p.min_p, 1.0)), kLeast) : kLeast;
    // buckets of even width from the largest down to what has a weight
    const float range = fminf(top - low, 30.5f * (float)fmin(temp, 1e30)), per = range > 0.0f ? (float)(BUCKETS - 1) / range : 0.0f;
    auto bucket_of = [&](float l) { return min((int)fminf((top - l) * per, (float)(BUCKETS - 1)), BUCKETS - 1); };

    // 2. the weights: of the whole row where a cut has to be found, else of what stays
    struct Weigh {
        Shared& s;
        const Weigher& weigh;
        const decltype(bucket_of)& bucket;
        double floor_x;
        bool by_value, count_too, mass_too;
        int lane;
        u64& sum;
        u64& all;
        __device__ void operator()(const float (&v)[4], int, int) const {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (v[e] == -INFINITY) continue;
                const bool weighs = v[e] >= weigh.least;
                if (by_value) {
                    const u64 w = mass_too && weighs ? weigh.fixed(weigh.log2w(v[e])) : 0;
                    const int b = bucket(v[e]);
                    if (count_too) atomicAdd(&s.cnt[b], 1u);
                    if (w) {
                        const unsigned lo = (unsigned)w, old = atomicAdd(&s.lo[b], lo);
                        const unsigned hi = (unsigned)(w >> 32) + (old + lo < lo);
                        if (hi) atomicAdd(&s.hi[b], hi);
                    }
                } else if (weighs) {
                    const double x = weigh.log2w(v[e]);
                    if (x >= floor_x) sum += weigh.fixed(x);
                }
            }
        }
        __device__ void done(int c) const {
            if (by_value) return;
            const u64 w = warp_sum(sum);
            all += w;
            sum = 0;
            if (lane == 0) s.chunk[c] = w;
        }
    };
    u64 lane_sum = 0, warp_all = 0;
    const bool by_value = cut_k || cut_p;
    over(row, begin, end, chunk, Weigh{s, weigh, bucket_of, floor_x, by_value, cut_k, cut_p, lane, lane_sum, warp_all});
    unsigned cut = 0;
    if (by_value) {
        sync();
        // each rank adds up its share of the buckets and hands it to all
        const int per_rank = BUCKETS / cs;
        for (int b = rank * per_rank + tid; b < (rank + 1) * per_rank; b += RT) {
            unsigned n = 0;
            u64 w = 0;
            for (int q = 0; q < cs; ++q) {
                n += *at(&s.cnt[b], q);
                w += (u64)*at(&s.hi[b], q) << 32;
                w += *at(&s.lo[b], q);
            }
            for (int q = 0; q < cs; ++q) { *at(&s.all_cnt[b], q) = n; *at(&s.all_mass[b], q) = w; }
        }
        sync();
        // two buckets a thread: what lies above them
        static_assert(BUCKETS == 2 * RT, "two buckets a thread");
        const unsigned n0 = s.all_cnt[2 * tid], n1 = s.all_cnt[2 * tid + 1];
        const u64 w0 = s.all_mass[2 * tid], w1 = s.all_mass[2 * tid + 1];
        unsigned n = n0 + n1;
        u64 w = w0 + w1;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned n2 = __shfl_up_sync(0xffffffffu, n, o);
            const u64 w2 = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) { n += n2; w += w2; }
        }
        if (lane == 31) { s.warp_n[warp] = n; s.warp_w[warp] = w; }
        if (tid == 0) { s.bucket = BUCKETS; s.wants = 0; }
        __syncthreads();
        u64 whole = 0;
        for (int q = 0; q < RW; ++q) {
            if (q < warp) { n += s.warp_n[q]; w += s.warp_w[q]; }
            whole += s.warp_w[q];
        }
        const double want = (double)p.top_p * (double)whole;
        auto reached = [&](u64 m) { return (double)m >= want; };
        // the first bucket (from the largest down) at whose end k ids, or the mass, are there
        unsigned an = n - n0 - n1;
        u64 aw = w - w0 - w1;
        int mine = BUCKETS;
#pragma unroll
        for (int i = 1; i >= 0; --i) {
            const unsigned bn = i ? n : n - n1;
            const u64 bw = i ? w : w - w1;
            const bool k = cut_k && bn >= (unsigned)p.top_k, m = cut_p && reached(bw);
            if (k || m) mine = 2 * tid + i;
        }
        if (mine < BUCKETS) atomicMin(&s.bucket, mine);
        __syncthreads();
        if (mine == s.bucket) {
            const int i = mine & 1;
            s.above_n = i ? an + n0 : an;
            s.above_w = i ? aw + w0 : aw;
            s.wants = (cut_k && (i ? n : n - n1) >= (unsigned)p.top_k ? 1 : 0) | (cut_p && reached(i ? w : w - w1) ? 2 : 0);
        }
        __syncthreads();
        const int bucket = s.bucket, wants = s.wants;
        if (bucket < BUCKETS) {
            // 3. the cut: the largest value of this bucket down to which k ids, or the mass, are there
            const unsigned above_n = s.above_n;
            const u64 above_w = s.above_w;
            auto enough = [&](unsigned k, u64 m) { return ((wants & 1) && above_n + k >= (unsigned)p.top_k) || ((wants & 2) && reached(above_w + m)); };
            bool listed = !cut_k || s.all_cnt[bucket] <= LIST;
            if (listed) {
                struct Gather {
                    Shared& s;
                    const Weigher& weigh;
                    const decltype(bucket_of)& bucket;
                    int* listed;
                    unsigned* keys;
                    u64* ws;
                    int which;
                    __device__ void operator()(const float (&v)[4], int, int) const {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (v[e] > -INFINITY && bucket(v[e]) == which) {
                                const int q = atomicAdd(listed, 1);
                                if (q >= LIST) continue;
                                keys[q] = logit_key(v[e]);
                                ws[q] = v[e] >= weigh.least ? weigh.fixed(weigh.log2w(v[e])) : 0;
                            }
                    }
                    __device__ void done(int) const {}
                };
                over(row, begin, end, chunk, Gather{s, weigh, bucket_of, at(&s.listed, 0), at(s.list_key, 0), at(s.list_w, 0), bucket});
                sync();
                listed = *at(&s.listed, 0) <= LIST;
                if (rank == 0 && listed) {
                    const int n = s.listed;
                    for (int i = tid; i < n; i += RT) {
                        const unsigned key = s.list_key[i];
                        unsigned ge = 0, gt = 0;
                        u64 wge = 0, wgt = 0;
                        for (int q = 0; q < n; ++q) {
                            const unsigned k = s.list_key[q];
                            const u64 x = s.list_w[q];
                            if (k >= key) { ++ge; wge += x; }
                            if (k > key) { ++gt; wgt += x; }
                        }
                        // all of a tie write the same
                        if (enough(ge, wge) && !(gt && enough(gt, wgt))) for (int q = 0; q < cs; ++q) *at(&s.cut, q) = key;
                    }
                }
                sync();
                cut = listed ? s.cut : 0;
            }
            if (!listed) {
                // more of them than the list holds: the cut's bits from the highest down, a pass each
                struct Count {
                    Shared& s;
                    const Weigher& weigh;
                    const decltype(bucket_of)& bucket;
                    int which;
                    unsigned cand;
                    unsigned& n;
                    u64& w;
                    bool mass_too;
                    __device__ void operator()(const float (&v)[4], int, int) const {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (v[e] > -INFINITY && logit_key(v[e]) >= cand && bucket(v[e]) == which) {
                                ++n;
                                if (mass_too && v[e] >= weigh.least) w += weigh.fixed(weigh.log2w(v[e]));
                            }
                    }
                    __device__ void done(int) const {}
                };
                for (int bit = 31; bit >= 0; --bit) {
                    const unsigned cand = cut | (1u << bit);
                    unsigned n = 0;
                    u64 w = 0;
                    over(row, begin, end, chunk, Count{s, weigh, bucket_of, bucket, cand, n, w, (wants & 2) != 0});
                    n = __reduce_add_sync(0xffffffffu, n);
                    w = warp_sum(w);
                    if (lane == 0) { s.warp_n[warp] = n; s.warp_w[warp] = w; }
                    __syncthreads();
                    if (tid == 0) {
                        for (int q = 1; q < RW; ++q) { n += s.warp_n[q]; w += s.warp_w[q]; }
                        s.wide_n = n; s.wide_w = w;
                    }
                    sync();
                    n = 0; w = 0;
                    for (int q = 0; q < cs; ++q) { n += *at(&s.wide_n, q); w += *at(&s.wide_w, q); }
                    if (n && enough(n, w)) cut = cand;
                    sync();
                }
            }
        }
        // the chunks' sums of what stays
        struct Keep {
            Shared& s;
            const Weigher& weigh;
            double floor_x;
            unsigned cut;
            int lane;
            u64& sum;
            u64& all;
            __device__ void operator()(const float (&v)[4], int, int) const {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (!(v[e] >= weigh.least) || logit_key(v[e]) < cut) continue;
                    const double x = weigh.log2w(v[e]);
                    if (x >= floor_x) sum += weigh.fixed(x);
                }
            }
            __device__ void done(int c) const {
                const u64 w = warp_sum(sum);
                all += w;
                sum = 0;
                if (lane == 0) s.chunk[c] = w;
            }
        };
        over(row, begin, end, chunk, Keep{s, weigh, floor_x, cut, lane, lane_sum, warp_all});
    }
    __syncthreads();                          // the warps' sums of the buckets have been read
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
            const float l = row.fix(__ldg(row.p + i));
            if (!(l >= weigh.least) || logit_key(l) < cut) return 0;
            const double x = weigh.log2w(l);
            return x >= floor_x ? weigh.fixed(x) : 0;
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
            if (prob) prob[r] = (float)(weigh.exact(weigh.log2w(row.fix(__ldg(row.p + i)))) * (double)(1ull << kFix) / (double)whole);
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
    if (device < 0 || device >= 64 || !ready[device]) {
        FC_TRY(select_device(device));
        FC_CUDA(cudaFuncSetAttribute(sample_rows_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(Shared)));
        if (device < 64) ready[device] = true;
    } else {
        int current = -1;
        FC_CUDA(cudaGetDevice(&current));
        if (current != device) FC_CUDA(cudaSetDevice(device));
    }
    // as many CTAs a row as are resident, each with 2048 ids at least
    int cs = 1, chunk = 128;
    while (cs < 8 && (long long)n_rows * cs * 2 <= 148 * 3 && (long long)cs * 2 * 2048 <= vocab) cs *= 2;
    while ((vocab + cs - 1) / cs > chunk * (CHUNKS - 1)) chunk *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)n_rows * cs);
    cfg.blockDim = dim3(RT);
    cfg.dynamicSmemBytes = sizeof(Shared);
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cs;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    FC_CUDA(cudaLaunchKernelEx(&cfg, sample_rows_kernel, logits, (long long)ld, vocab, params, u, token, prob, cs, chunk));
    FC_LAUNCHED();
    return FC_OK;
}
