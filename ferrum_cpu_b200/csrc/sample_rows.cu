// Draws from rows of logits on the device with given random numbers: temperature -> top-k -> top-p -> min-p -> the first id at which
// the running mass of what stays reaches u times its whole. The filters are those of sample.cu (all of a tie at a cut stays), and each of them
// keeps what lies above a value of its own: top-k the k-th largest logit, top-p the largest logit down to which the mass reaches
// top_p of the whole row, min-p the logit whose weight is min_p of the largest. They therefore commute.
//
// Weights are exp((l - max) / T) in 64 bits: a flat row of 2^17 ids has borders 2^-17 apart, of which sums in 32 bits miss one
// in a hundred.
#include "fc_common.cuh"

namespace fc {

namespace {

constexpr int RT = 512;
constexpr double kLeast = 9.094947017729282e-13;   // 2^-40: weights under it are not drawn

// Logits in their order as unsigned keys; NaN is the least and stands for a forbidden id, as -inf.
__device__ __forceinline__ unsigned logit_key(float l) {
    l += 0.0f;
    const unsigned b = __float_as_uint(l);
    return l != l ? 0u : b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}

template <class T, class Op>
__device__ T block_reduce(T v, T* red, const Op& op) {
    for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = red[0];
    for (int w = 1; w < RT / 32; ++w) v = op(v, red[w]);
    return v;
}

__global__ void __launch_bounds__(RT) sample_rows_kernel(const float* __restrict__ logits, long long ld, int V, const fc_row_sampling* __restrict__ params,
                                                         const float* __restrict__ u, int* __restrict__ token, float* __restrict__ prob) {
    __shared__ double redd[RT / 32];
    __shared__ float redf[RT / 32];
    __shared__ int redi[RT / 32];
    const int tid = threadIdx.x;
    const float* row = logits + (size_t)blockIdx.x * ld;
    const fc_row_sampling p = params[blockIdx.x];
    auto sum = [](auto x, auto y) { return x + y; };
    auto least = [](int x, int y) { return min(x, y); };
    float best = -INFINITY;
    for (int i = tid; i < V; i += RT) best = fmaxf(best, row[i]);
    best = block_reduce(best, redf, [](float x, float y) { return fmaxf(x, y); });
    if (best == -INFINITY) {                          // nothing can be drawn
        if (tid == 0) { token[blockIdx.x] = -1; if (prob) prob[blockIdx.x] = 0.0f; }
        return;
    }
    if (!(p.temperature > 0.0f)) {
        int at = V;
        for (int i = tid; i < V && at == V; i += RT) if (row[i] == best) at = i;
        at = block_reduce(at, redi, least);
        if (tid == 0) { token[blockIdx.x] = at; if (prob) prob[blockIdx.x] = 1.0f; }
        return;
    }
    const double t = fmax((double)p.temperature, 0.01);
    auto weight = [&](float l) { return l == best ? 1.0 : l == l ? exp(((double)l - (double)best) / t) : 0.0; };
    unsigned cut = 0;
    if (p.top_k > 0 && p.top_k < V)
        for (int bit = 31; bit >= 0; --bit) {
            const unsigned cand = cut | (1u << bit);
            int n = 0;
            for (int i = tid; i < V; i += RT) n += logit_key(row[i]) >= cand;
            if (block_reduce(n, redi, sum) >= p.top_k) cut = cand;
        }
    if (p.top_p < 1.0f) {
        double all = 0.0;
        for (int i = tid; i < V; i += RT) all += weight(row[i]);
        const double want = (double)p.top_p * block_reduce(all, redd, sum);
        unsigned c = 0;
        for (int bit = 31; bit >= 0; --bit) {
            const unsigned cand = c | (1u << bit);
            if (cand > logit_key(best)) continue;     // the largest always stays
            double m = 0.0;
            for (int i = tid; i < V; i += RT) m += logit_key(row[i]) >= cand ? weight(row[i]) : 0.0;
            if (block_reduce(m, redd, sum) >= want) c = cand;
        }
        cut = max(cut, c);
    }
    const double floor_w = p.min_p > 0.0f ? fmin((double)p.min_p, 1.0) : 0.0;
    auto stays = [&](float l, double w) { return logit_key(l) >= cut && w >= floor_w && w >= kLeast; };
    // thread t owns the ids [t * chunk, ..)
    const int chunk = (V + RT - 1) / RT, i0 = min(tid * chunk, V), i1 = min(i0 + chunk, V);
    double mine = 0.0;
    for (int i = i0; i < i1; ++i) {
        const double w = weight(row[i]);
        if (stays(row[i], w)) mine += w;
    }
    __shared__ double before[RT + 1];
    before[tid + 1] = mine;
    __syncthreads();
    if (tid == 0) {
        before[0] = 0.0;
        for (int q = 0; q < RT; ++q) before[q + 1] += before[q];
    }
    __syncthreads();
    const double whole = before[RT], r = (double)u[blockIdx.x] * whole;
    double cum = before[tid];
    int at = V, last = -1;
    for (int i = i0; i < i1; ++i) {
        const double w = weight(row[i]);
        if (!stays(row[i], w)) continue;
        cum += w;
        last = i;
        if (at == V && cum >= r) at = i;
    }
    at = block_reduce(at, redi, least);
    last = block_reduce(last, redi, [](int x, int y) { return max(x, y); });
    if (at == V) at = last;                           // u of 1, or a rounding
    if (tid == 0) { token[blockIdx.x] = at; if (prob) prob[blockIdx.x] = (float)(weight(row[at]) / whole); }
}

}  // namespace
}  // namespace fc

using namespace fc;

extern "C" int fc_sample_rows_dev(int device, const float* logits, int64_t ld, int n_rows, int vocab, const fc_row_sampling* params, const float* u,
                                  int32_t* token, float* prob, void* stream) {
    if (!logits || !params || !u || !token) return fail(FC_E_ARG, "fc_sample_rows_dev: null argument");
    if (n_rows < 0 || vocab <= 0 || vocab > (1 << 24) || ld < vocab) return fail(FC_E_SHAPE, "fc_sample_rows_dev: %d rows of %d logits, %lld apart", n_rows, vocab, (long long)ld);
    if (!aligned16(params)) return fail(FC_E_ARG, "fc_sample_rows_dev: params must be 16-byte aligned");
    if (!n_rows) return FC_OK;
    FC_TRY(select_device(device));
    sample_rows_kernel<<<n_rows, RT, 0, (cudaStream_t)stream>>>(logits, ld, vocab, params, u, token, prob);
    FC_LAUNCHED();
    return FC_OK;
}
