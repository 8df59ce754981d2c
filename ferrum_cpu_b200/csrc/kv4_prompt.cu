// Attention of many query rows over the cache of 4-bit levels (layout: kv4.cuh), and the weights that positions receive from them.
//
// kv4_prompt_kernel: a CTA takes 128 query columns (rows x heads that share a key / value head), 16 a warp, and passes over tiles of 64
// positions with a running maximum and sum. The CTA turns a tile's levels into f16 fragments in shared memory once for all its
// warps. S = q K^T: exact levels against two f16 planes of q, a block's sum times its scale in f32. O = P V: exact levels against two
// planes of the weight times the value's scale. That product is formed in f16 pairs: with p = ph + pl, the high plane is
// rn(ph d) and the low one (ph d - rn(ph d), exact in a fused multiply-add) + pl d. So that it stays within f16, a position's scales are
// divided by the power of two 2^e of the largest of its blocks (and times 2^kScaleLift), and e is added to its score: the running maximum is that of s + e, and
// the sum takes 2^-e back. Sums of products start from zero in every tile and are added to the row's in f32, because
// the tensor core truncates.
//
// kv4_weights_kernel: the transposed walk. A warp keeps 32 positions' levels in registers (16 of heads
// above 128) and passes over all columns, whose
// maximum and sum the attention has left; each position is added up by one warp in one order.
//
// Bound: the latencies of products and what depends on them, of which two warps a scheduler cover about half: 1.46 instructions a cycle, the tensor
// pipe 53 % busy, most stalls fixed waits behind an instruction. mma.sync reaches 550 TFLOP/s alone, and 460 with three other instructions to a product;
// here there are four to six. 6007 rows of 32 heads of 128: 2.06 ms, 144 TFLOP/s, executed twice. 2048 rows of 32 heads of 64: 146 us, their weights
// 98 (the same with 64 positions a warp); of 128: 269 and 191.
// One CTA of 8 warps an SM at 255 registers; two or three CTAs, or 12 warps with q in shared memory, are no faster. Heads above 128: 4 warps with q in
// shared memory, and registers that spill (40 bytes at 160, 128 at 192, 448 at 224, 1248 at 256): 2048 rows of 32 heads of 160 493 us, of 192 603, of 256 951.
#include <cooperative_groups.h>

#include <climits>

#include "kv4_frag.cuh"

namespace fc {

namespace {

namespace cg = cooperative_groups;

constexpr int KT = 64;                           // positions a tile

template <int NB>
struct PromptShape {
    static constexpr int WARPS = NB <= 4 ? 8 : 4;
    static constexpr int COLS = 16 * WARPS, DIM = NB * kKvBlock, PAD = DIM + 4;
    static constexpr int KBYTES = NB * 4096, VBYTES = NB * 4096;                       // levels as fragments
    static constexpr int KD = KBYTES + VBYTES, VD = KD + NB * KT * 4, EX = VD + NB * KT * 2, BYTES = EX + KT * 8;   // scales; {e, 2^-e}
    static constexpr bool QS = NB > 4;           // q in shared memory
    static constexpr int QBYTES = QS ? COLS * DIM * 4 : 0;
    static constexpr int JOIN = COLS * PAD * 4;
    static constexpr int SMEM = QBYTES + (2 * BYTES > JOIN ? 2 * BYTES : JOIN);
    static constexpr int CTAS = 1;
};

// Channels 32 b + 8 t .. + 7 of two rows of q (rows g and g + 8 of 16), as they are; zeros for a row that is none.
template <int NB>
__device__ __forceinline__ void query_ask(const float* q0, const float* q1, float4 (&x)[2][NB][2]) {
    const float4 zero = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const float* q = r ? q1 : q0;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int u = 0; u < 2; ++u) x[r][b][u] = q ? *(const float4*)(q + 32 * b + 4 * u) : zero;
    }
}
// As fragments of two planes, brought to [2^13, 2^14) by a power of two a row, whose inverses come back in inv. Registers 4 u + {0: row g,
// 1: row g + 8} of a block hold the nibbles 2 u, {2, 3} the nibbles 2 u + 1.
template <int NB>
__device__ __forceinline__ void query_planes(const float4 (&x)[2][NB][2], float scale, uint32_t (&qh)[NB][8], uint32_t (&ql)[NB][8], float (&inv)[2]) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        float top = 0.0f;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const float4 v = x[r][b][u];
                top = fmaxf(fmaxf(top, fmaxf(fabsf(v.x * scale), fabsf(v.y * scale))), fmaxf(fabsf(v.z * scale), fabsf(v.w * scale)));
            }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int shift = plane_shift(top);
        const float up = exp2i(shift);
        inv[r] = exp2i(-shift);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const float4 lo = x[r][b][0], hi = x[r][b][1];
            const float v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
            for (int j = 0; j < 4; ++j)
                planes_of(v[j] * scale * up, v[j + 4] * scale * up, &qh[b][4 * (j >> 1) + 2 * (j & 1) + r], &ql[b][4 * (j >> 1) + 2 * (j & 1) + r]);
        }
    }
}

// A tile of the cache on its way: what a thread brings of it.
template <int NB, int PASS>
struct RawTile {
    uint32_t k[PASS][NB], v[PASS][NB];
    __half d[NB];
};
template <int NB, int PASS>
__device__ __forceinline__ void tile_ask(const Kv4& c, size_t row, int tid, RawTile<NB, PASS>& r) {
    const int lane = tid & 31;
#pragma unroll
    for (int p = 0; p < PASS; ++p) {
        const int e = tid + p * (256 / PASS), w = e >> 5;
        load_words(c.kq + row * (NB * 4) + e * NB, r.k[p]);
        // lane = t + 4 (g & 1) + 8 (pair / 4 & 1) + 16 (g >> 1 & 1), warp = (g >> 2) + 2 (pair / 8)
        const int g = (lane >> 2 & 1) | (lane >> 4) << 1 | (w & 1) << 2, pair = (lane & 3) + 4 * (lane >> 3 & 1) + 8 * (w >> 1);
        load_words(c.vq + row * (NB * 4) + (pair * 8 + g) * NB, r.v[p]);
    }
    const __half* d = tid < KT ? c.kd + (row + tid) * NB : c.vd + (row + (tid & (KT - 1))) * NB;
    if (tid < 2 * KT)
#pragma unroll
        for (int b = 0; b < NB; ++b) r.d[b] = d[b];
}
template <int NB, int PASS>
__device__ __forceinline__ void tile_lay(char* buf, int tid, const RawTile<NB, PASS>& r) {
    using S = PromptShape<NB>;
    const int lane = tid & 31;
#pragma unroll
    for (int p = 0; p < PASS; ++p) {
        const int e = tid + p * (256 / PASS), w = e >> 5;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            uint32_t f[4];
            levels_of(r.k[p][b], f);
            // word t of position 8 n + g: the lane that reads it is its own; n = warp
            ((uint4*)buf)[(b * 8 + w) * 32 + lane] = make_uint4(f[0], f[1], f[2], f[3]);
        }
        const int g = (lane >> 2 & 1) | (lane >> 4) << 1 | (w & 1) << 2, odd = lane >> 3 & 1;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            uint32_t f[4];
            levels_of(r.v[p][b], f);
            // pairs t and t + 4 of 16 positions meet: the first keeps channels 8 j + g of j = 0, 1, the other those of j = 2, 3
            const uint32_t x = __shfl_xor_sync(0xffffffffu, odd ? f[0] : f[2], 8), y = __shfl_xor_sync(0xffffffffu, odd ? f[1] : f[3], 8);
            const uint4 out = odd ? make_uint4(x, f[2], y, f[3]) : make_uint4(f[0], x, f[1], y);
            ((uint4*)(buf + S::KBYTES))[((b * 4 + (w >> 1)) * 2 + odd) * 32 + g * 4 + (lane & 3)] = out;
        }
    }
    if (tid < KT) {
#pragma unroll
        for (int b = 0; b < NB; ++b) ((float*)(buf + S::KD))[b * KT + tid] = __half2float(r.d[b]);
    } else if (tid < 2 * KT) {
        const int j = tid - KT;
        float d[NB], top = 0.0f;
#pragma unroll
        for (int b = 0; b < NB; ++b) { d[b] = __half2float(r.d[b]); top = fmaxf(top, fabsf(d[b])); }
        // an f16 above 0 is a normal f32, of 2^-24 at least. Zeros bring nothing to the sums of products and must not hold the maximum that the
        // others' planes are scaled by: seven powers of two below the least of them, which rounds a score no more than that does
        const int e = top > 0.0f ? (__float_as_int(top) >> 23) - 127 : -31;
        const float back = exp2i(-e);
#pragma unroll
        for (int b = 0; b < NB; ++b) ((__half*)(buf + S::VD))[b * KT + j] = __float2half_rn(d[b] * back * (float)(1 << kScaleLift));
        ((float2*)(buf + S::EX))[j] = make_float2((float)e, back);
    }
}

template <int NB>
__global__ void __launch_bounds__(32 * PromptShape<NB>::WARPS, PromptShape<NB>::CTAS)
kv4_prompt_kernel(Kv4 c, Kv4Attend a, KvRows rows, int cs, float2* __restrict__ stats) {
    using S = PromptShape<NB>;
    constexpr int WARPS = S::WARPS, DIM = S::DIM, PAD = S::PAD, THREADS = 32 * WARPS, PASS = 8 / WARPS;
    extern __shared__ __align__(16) char smem[];
    __shared__ float2 ml[S::COLS];
    pdl_trigger();
    pdl_wait();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int rank = blockIdx.x % cs, h = blockIdx.x / cs % c.n_kv, seq = blockIdx.z;
    const int first = rows.start[seq], n = rows.start[seq + 1] - first, all_cols = n * a.group;
    // the last columns, of all heads, see most: they go first
    const unsigned share = cs * c.n_kv;
    const int col0 = (int)(gridDim.x / share - 1 - blockIdx.x / share) * S::COLS, cols = min(all_cols - col0, S::COLS);
    if (cols <= 0) return;                       // the whole cluster
    const int len = a.lens[seq], end = a.k ? len + n : len;
    float* const out = a.out + (size_t)first * a.ldo + (size_t)h * a.group * DIM;
    auto place = [&](int col) { const int i = (col0 + col) / a.group; return (size_t)i * a.ldo + ((col0 + col) - i * a.group) * DIM; };
    if (len < 0 || len > c.cap - (a.k ? n : 0)) {
        for (int e = rank * THREADS + tid; e < cols * DIM; e += cs * THREADS) out[place(e / DIM) + e % DIM] = __int_as_float(0x7fffffff);
        return;
    }
    const int base = end - n + 1;                // row i sees the positions below base + i
    auto sees = [&](int col) { return col < cols ? max(0, base + (col0 + col) / a.group) : 0; };
    const int tiles = (max(0, base + (col0 + cols - 1) / a.group) + KT - 1) / KT;
    const size_t row0 = c.row(seq, h, 0);
    char* const bufs = smem + S::QBYTES;

    RawTile<NB, PASS> raw;
    if (rank < tiles) tile_ask<NB, PASS>(c, row0 + (size_t)rank * KT, tid, raw);

    const int ca = warp * 16 + g, cb = ca + 8;    // this lane's two columns
    uint32_t qh[NB][8], ql[NB][8];
    float inv[2];
    {
        auto from = [&](int col) {
            const int i = (col0 + col) / a.group, head = h * a.group + (col0 + col) - i * a.group;
            return col < cols ? a.q + (size_t)(first + i) * a.ldq + (size_t)head * DIM + 8 * t : nullptr;
        };
        float4 x[2][NB][2];
        query_ask<NB>(from(ca), from(cb), x);
        query_planes<NB>(x, a.scale * 1.44269504f, qh, ql, inv);
    }
    uint4* const qs = (uint4*)smem + warp * (NB * 4 * 32) + lane;     // [block][plane, fragment][lane]
    if (S::QS) {
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                qs[(b * 4 + u) * 32] = make_uint4(qh[b][4 * u], qh[b][4 * u + 1], qh[b][4 * u + 2], qh[b][4 * u + 3]);
                qs[(b * 4 + 2 + u) * 32] = make_uint4(ql[b][4 * u], ql[b][4 * u + 1], ql[b][4 * u + 2], ql[b][4 * u + 3]);
            }
    }
    const int seen_a = sees(ca), seen_b = sees(cb);
    const int warp_first = warp * 16 < cols ? max(0, base + (col0 + warp * 16) / a.group) : 0;
    const int warp_last = warp * 16 < cols ? max(0, base + (col0 + min(cols, warp * 16 + 16) - 1) / a.group) : 0;

    float o[NB][4][4] = {}, ma = -INFINITY, mb = -INFINITY, la = 0.0f, lb = 0.0f;
    int flip = 0;
    if (rank < tiles) tile_lay<NB, PASS>(bufs, tid, raw);
    __syncthreads();
    for (int tile = rank; tile < tiles; tile += cs) {
        const char* buf = bufs + flip * S::BYTES;
        if (tile + cs < tiles) tile_ask<NB, PASS>(c, row0 + (size_t)(tile + cs) * KT, tid, raw);
        const int j0 = tile * KT;
        if (j0 < warp_last) {
            float s[8][4];
            const float* kd = (const float*)(buf + S::KD);
            constexpr int NG = 4;                 // tiles of 8 positions side by side: four products between two of one sum
#pragma unroll
            for (int n0 = 0; n0 < 8; n0 += NG) {
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    uint32_t h0[4], h1[4], r0[4], r1[4];
                    if (S::QS) {
                        const uint4 x0 = qs[(b * 4) * 32], x1 = qs[(b * 4 + 1) * 32], y0 = qs[(b * 4 + 2) * 32], y1 = qs[(b * 4 + 3) * 32];
                        h0[0] = x0.x; h0[1] = x0.y; h0[2] = x0.z; h0[3] = x0.w; h1[0] = x1.x; h1[1] = x1.y; h1[2] = x1.z; h1[3] = x1.w;
                        r0[0] = y0.x; r0[1] = y0.y; r0[2] = y0.z; r0[3] = y0.w; r1[0] = y1.x; r1[1] = y1.y; r1[2] = y1.z; r1[3] = y1.w;
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) { h0[e] = qh[b][e]; h1[e] = qh[b][4 + e]; r0[e] = ql[b][e]; r1[e] = ql[b][4 + e]; }
                    }
                    uint4 f[NG];
                    float x[NG][4] = {};
#pragma unroll
                    for (int i = 0; i < NG; ++i) f[i] = ((const uint4*)buf)[(b * 8 + n0 + i) * 32 + lane];
#pragma unroll
                    for (int i = 0; i < NG; ++i) mma16816(x[i], r0, f[i].x, f[i].y);
#pragma unroll
                    for (int i = 0; i < NG; ++i) mma16816(x[i], r1, f[i].z, f[i].w);
#pragma unroll
                    for (int i = 0; i < NG; ++i) mma16816(x[i], h0, f[i].x, f[i].y);
#pragma unroll
                    for (int i = 0; i < NG; ++i) mma16816(x[i], h1, f[i].z, f[i].w);
#pragma unroll
                    for (int i = 0; i < NG; ++i) {
                        const float2 d = *(const float2*)(kd + b * KT + 8 * (n0 + i) + 2 * t);
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[n0 + i][e] = b ? fmaf(x[i][e], e & 1 ? d.y : d.x, s[n0 + i][e]) : x[i][e] * (e & 1 ? d.y : d.x);
                    }
                }
            }
            const float2* ex = (const float2*)(buf + S::EX);
            float ta = -INFINITY, tb = -INFINITY;
            if (j0 + KT <= warp_first) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float4 e = *(const float4*)(ex + 8 * i + 2 * t);
                    s[i][0] = fmaf(s[i][0], inv[0], e.x);
                    s[i][1] = fmaf(s[i][1], inv[0], e.z);
                    s[i][2] = fmaf(s[i][2], inv[1], e.x);
                    s[i][3] = fmaf(s[i][3], inv[1], e.z);
                    ta = fmaxf(ta, fmaxf(s[i][0], s[i][1]));
                    tb = fmaxf(tb, fmaxf(s[i][2], s[i][3]));
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float4 e = *(const float4*)(ex + 8 * i + 2 * t);
                    const int j = j0 + 8 * i + 2 * t;
                    s[i][0] = j < seen_a ? fmaf(s[i][0], inv[0], e.x) : -INFINITY;
                    s[i][1] = j + 1 < seen_a ? fmaf(s[i][1], inv[0], e.z) : -INFINITY;
                    s[i][2] = j < seen_b ? fmaf(s[i][2], inv[1], e.x) : -INFINITY;
                    s[i][3] = j + 1 < seen_b ? fmaf(s[i][3], inv[1], e.z) : -INFINITY;
                    ta = fmaxf(ta, fmaxf(s[i][0], s[i][1]));
                    tb = fmaxf(tb, fmaxf(s[i][2], s[i][3]));
                }
            }
            ta = fmaxf(ta, __shfl_xor_sync(0xffffffffu, ta, 1));
            tb = fmaxf(tb, __shfl_xor_sync(0xffffffffu, tb, 1));
            ta = fmaxf(fmaxf(ta, __shfl_xor_sync(0xffffffffu, ta, 2)), ma);
            tb = fmaxf(fmaxf(tb, __shfl_xor_sync(0xffffffffu, tb, 2)), mb);
            const float za = (ta == -INFINITY ? 0.0f : ta) - kLift, zb = (tb == -INFINITY ? 0.0f : tb) - kLift;
            if (__any_sync(0xffffffffu, ta != ma || tb != mb)) {
                const float fa = ex2(ma - kLift - za), fb = ex2(mb - kLift - zb);
                la *= fa; lb *= fb;
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int j = 0; j < 4; ++j) { o[b][j][0] *= fa; o[b][j][1] *= fa; o[b][j][2] *= fb; o[b][j][3] *= fb; }
                ma = ta; mb = tb;
            }
            uint32_t ph[4][4], pl[4][4];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float4 e = *(const float4*)(ex + 8 * i + 2 * t);
                const float p0 = ex2(s[i][0] - za), p1 = ex2(s[i][1] - za), p2 = ex2(s[i][2] - zb), p3 = ex2(s[i][3] - zb);
                la = fmaf(p0, e.y, la); la = fmaf(p1, e.w, la);
                lb = fmaf(p2, e.y, lb); lb = fmaf(p3, e.w, lb);
                planes_of(p0, p1, &ph[i >> 1][2 * (i & 1)], &pl[i >> 1][2 * (i & 1)]);
                planes_of(p2, p3, &ph[i >> 1][2 * (i & 1) + 1], &pl[i >> 1][2 * (i & 1) + 1]);
            }
            const char* vd = buf + S::VD;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                float x[4][4] = {};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint32_t d0 = *(const uint32_t*)(vd + (b * KT + 16 * k + 2 * t) * 2), d1 = *(const uint32_t*)(vd + (b * KT + 16 * k + 8 + 2 * t) * 2);
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t d = e < 2 ? d0 : d1;
                        hi[e] = hmul2u(ph[k][e], d);
                        lo[e] = hfma2u(pl[k][e], d, hfms2u(ph[k][e], d, hi[e]));
                    }
                    const uint4* vf = (const uint4*)(buf + S::KBYTES) + (b * 4 + k) * 64 + lane;
                    const uint4 v0 = vf[0], v1 = vf[32];
                    mma16816(x[0], lo, v0.x, v0.y);
                    mma16816(x[1], lo, v0.z, v0.w);
                    mma16816(x[2], lo, v1.x, v1.y);
                    mma16816(x[3], lo, v1.z, v1.w);
                    mma16816(x[0], hi, v0.x, v0.y);
                    mma16816(x[1], hi, v0.z, v0.w);
                    mma16816(x[2], hi, v1.x, v1.y);
                    mma16816(x[3], hi, v1.z, v1.w);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[b][j][e] += x[j][e];
            }
        }
        flip ^= 1;
        if (tile + cs < tiles) tile_lay<NB, PASS>(bufs + flip * S::BYTES, tid, raw);
        __syncthreads();
    }
    la += __shfl_xor_sync(0xffffffffu, la, 1);
    lb += __shfl_xor_sync(0xffffffffu, lb, 1);
    la += __shfl_xor_sync(0xffffffffu, la, 2);
    lb += __shfl_xor_sync(0xffffffffu, lb, 2);
    auto stat = [&](int col) -> float2& {
        const int i = (col0 + col) / a.group;
        return stats[((size_t)first + i) * (c.n_kv * a.group) + h * a.group + (col0 + col) - i * a.group];
    };
    if (cs == 1) {
        const float one = 1.0f / (float)(1 << kScaleLift), fa = la == 0.0f ? 0.0f : one / la, fb = lb == 0.0f ? 0.0f : one / lb;
        if (ca < cols) {
            float* to = out + place(ca) + 2 * t;
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int j = 0; j < 4; ++j) *(float2*)(to + 32 * b + 8 * j) = make_float2(o[b][j][0] * fa, o[b][j][1] * fa);
            if (t == 0 && stats) stat(ca) = make_float2(ma == -INFINITY ? 0.0f : ma - kLift, la);
        }
        if (cb < cols) {
            float* to = out + place(cb) + 2 * t;
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int j = 0; j < 4; ++j) *(float2*)(to + 32 * b + 8 * j) = make_float2(o[b][j][2] * fb, o[b][j][3] * fb);
            if (t == 0 && stats) stat(cb) = make_float2(mb == -INFINITY ? 0.0f : mb - kLift, lb);
        }
        return;
    }
    // the ranks' shares of the positions meet: [column][channel] in every rank's shared memory
    float* const part = (float*)bufs;
    if (t == 0) { ml[ca] = make_float2(ma, la); ml[cb] = make_float2(mb, lb); }
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            *(float2*)(part + ca * PAD + 32 * b + 8 * j + 2 * t) = make_float2(o[b][j][0], o[b][j][1]);
            *(float2*)(part + cb * PAD + 32 * b + 8 * j + 2 * t) = make_float2(o[b][j][2], o[b][j][3]);
        }
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    for (int e = rank * THREADS + tid; e < cols * (DIM / 4); e += cs * THREADS) {
        const int col = e / (DIM / 4), ch = e % (DIM / 4) * 4;
        float m = -INFINITY, l = 0.0f;
        for (int r = 0; r < cs; ++r) m = fmaxf(m, cluster.map_shared_rank(ml, r)[col].x);
        const float z = m == -INFINITY ? 0.0f : m;
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int r = 0; r < cs; ++r) {
            const float2 y = cluster.map_shared_rank(ml, r)[col];
            const float f = ex2(y.x - z);
            const float4 v = *(const float4*)(cluster.map_shared_rank(part, r) + col * PAD + ch);
            l = fmaf(y.y, f, l);
            x.x = fmaf(v.x, f, x.x); x.y = fmaf(v.y, f, x.y); x.z = fmaf(v.z, f, x.z); x.w = fmaf(v.w, f, x.w);
        }
        const float f = l == 0.0f ? 0.0f : 1.0f / (float)(1 << kScaleLift) / l;
        *(float4*)(out + place(col) + ch) = make_float4(x.x * f, x.y * f, x.z * f, x.w * f);
        if (ch == 0 && stats) stat(col) = make_float2(m == -INFINITY ? 0.0f : m - kLift, l);
    }
    cluster.sync();                              // no rank leaves while another reads its memory
}

// ---- the weights that positions receive --------------------------------------------------------------------------
constexpr int WW = 4, WCOLS = 16 * WW;           // warps; columns a pass
template <int NB>
struct WeightsShape {
    static constexpr int TILES = NB <= 4 ? 4 : 2, POS = 8 * TILES * WW;      // tiles of 8 positions a warp, positions a CTA
    static constexpr int BUFS = NB <= 4 ? 2 : 1, BUF = WW * NB * 4 * 512 + WCOLS * 16, SMEM = BUFS * BUF;
};

template <int NB>
__global__ void __launch_bounds__(32 * WW) kv4_weights_kernel(Kv4 c, Kv4Attend a, KvRows rows, int cs, const float2* __restrict__ stats) {
    using S = WeightsShape<NB>;
    constexpr int DIM = NB * kKvBlock, TILES = S::TILES, BUFS = S::BUFS;
    extern __shared__ __align__(16) char smem[]; // [buffer]: fragments [16 columns][block, plane and fragment][lane], columns
    __shared__ float part[S::POS];
    pdl_trigger();
    pdl_wait();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3, rank = blockIdx.x % cs, h = blockIdx.x / cs % c.n_kv, seq = blockIdx.z;
    const int first = rows.start[seq], n = rows.start[seq + 1] - first, all_cols = n * a.group;
    const int len = a.lens[seq], end = a.k ? len + n : len;
    const int j00 = blockIdx.x / (cs * c.n_kv) * S::POS, j0 = j00 + warp * (8 * TILES), base = end - n + 1;
    if (n == 0 || len < 0 || len > c.cap - (a.k ? n : 0) || j00 >= end) return;      // the whole cluster
    // levels and scales of the warp's positions
    uint32_t kf[TILES][NB][4];
    float2 kd[TILES][NB];
#pragma unroll
    for (int i = 0; i < TILES; ++i) {
        const size_t row = c.row(seq, h, 0) + min(j0, c.cap_pad - 8 * TILES) + 8 * i;
        uint32_t w[NB];
        load_words(c.kq + (row + g) * (NB * 4) + t * NB, w);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            levels_of(w[b], kf[i][b]);
            kd[i][b] = make_float2(__half2float(c.kd[(row + 2 * t) * NB + b]), __half2float(c.kd[(row + 2 * t + 1) * NB + b]));
        }
    }
    float sum[TILES][2] = {};
    // the first column that sees any of the CTA's positions; the ranks take turns
    const int col_first = min(n, max(0, j00 + 1 - base)) * a.group / WCOLS * WCOLS;
    auto from = [&](int col) {
        const int i = col / a.group, head = h * a.group + col - i * a.group;
        return col < all_cols ? a.q + (size_t)(first + i) * a.ldq + (size_t)head * DIM + 8 * t : nullptr;
    };
    float4 raw[2][NB][2];
    int c0 = col_first + rank * WCOLS;
    if (BUFS == 2 && c0 < all_cols) query_ask<NB>(from(c0 + warp * 16 + g), from(c0 + warp * 16 + g + 8), raw);
    int flip = 0;
    for (; c0 < all_cols; c0 += cs * WCOLS) {
        char* const buf = smem + flip * S::BUF;
        uint4* const qf = (uint4*)buf;
        float4* const col_of = (float4*)(buf + WW * NB * 4 * 512);     // 1 / power of two of q, maximum, 1 / sum, positions seen
        {
            // every warp lays 16 columns
            const int ca = c0 + warp * 16 + g;
            uint32_t qh[NB][8], ql[NB][8];
            float inv[2];
            if (BUFS == 1) query_ask<NB>(from(ca), from(ca + 8), raw);
            query_planes<NB>(raw, a.scale * 1.44269504f, qh, ql, inv);
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    qf[(warp * (NB * 4) + b * 4 + u) * 32 + lane] = make_uint4(qh[b][4 * u], qh[b][4 * u + 1], qh[b][4 * u + 2], qh[b][4 * u + 3]);
                    qf[(warp * (NB * 4) + b * 4 + 2 + u) * 32 + lane] = make_uint4(ql[b][4 * u], ql[b][4 * u + 1], ql[b][4 * u + 2], ql[b][4 * u + 3]);
                }
            if (t == 0)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const int col = ca + 8 * r, i = col / a.group;
                    float2 st = make_float2(0.0f, 0.0f);
                    if (col < all_cols) st = stats[((size_t)first + i) * (c.n_kv * a.group) + h * a.group + col - i * a.group];
                    col_of[warp * 16 + 8 * r + g] = make_float4(inv[r], st.x, st.y == 0.0f ? 0.0f : 1.0f / st.y, __int_as_float(col < all_cols ? base + i : 0));
                }
            const int next = ca + cs * WCOLS;
            if (BUFS == 2 && c0 + cs * WCOLS < all_cols) query_ask<NB>(from(next), from(next + 8), raw);
        }
        __syncthreads();                         // with two buffers, the next pass's columns are laid while this one's are read
#pragma unroll 1
        for (int q = 0; q < WW; ++q) {
            const float4 xa = col_of[q * 16 + g], xb = col_of[q * 16 + g + 8];
            const int seen_a = __float_as_int(xa.w), seen_b = __float_as_int(xb.w);
            float s[TILES][4];
#pragma unroll
            for (int i = 0; i < TILES; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[i][e] = 0.0f;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const uint4* f = qf + (q * (NB * 4) + b * 4) * 32 + lane;
                const uint4 x0 = f[0], x1 = f[32], y0 = f[64], y1 = f[96];
                const uint32_t h0[4] = {x0.x, x0.y, x0.z, x0.w}, h1[4] = {x1.x, x1.y, x1.z, x1.w}, r0[4] = {y0.x, y0.y, y0.z, y0.w}, r1[4] = {y1.x, y1.y, y1.z, y1.w};
#pragma unroll
                for (int i = 0; i < TILES; ++i) {
                    float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    mma16816(x, r0, kf[i][b][0], kf[i][b][1]);
                    mma16816(x, r1, kf[i][b][2], kf[i][b][3]);
                    mma16816(x, h0, kf[i][b][0], kf[i][b][1]);
                    mma16816(x, h1, kf[i][b][2], kf[i][b][3]);
                    s[i][0] = fmaf(x[0], kd[i][b].x, s[i][0]);
                    s[i][1] = fmaf(x[1], kd[i][b].y, s[i][1]);
                    s[i][2] = fmaf(x[2], kd[i][b].x, s[i][2]);
                    s[i][3] = fmaf(x[3], kd[i][b].y, s[i][3]);
                }
            }
            if (__all_sync(0xffffffffu, min(seen_a, seen_b) >= j0 + 8 * TILES)) {
#pragma unroll
                for (int i = 0; i < TILES; ++i) {
                    sum[i][0] = fmaf(ex2(fmaf(s[i][0], xa.x, -xa.y)), xa.z, fmaf(ex2(fmaf(s[i][2], xb.x, -xb.y)), xb.z, sum[i][0]));
                    sum[i][1] = fmaf(ex2(fmaf(s[i][1], xa.x, -xa.y)), xa.z, fmaf(ex2(fmaf(s[i][3], xb.x, -xb.y)), xb.z, sum[i][1]));
                }
            } else {
#pragma unroll
                for (int i = 0; i < TILES; ++i) {
                    const int j = j0 + 8 * i + 2 * t;
                    sum[i][0] += (j < seen_a ? ex2(fmaf(s[i][0], xa.x, -xa.y)) * xa.z : 0.0f) + (j < seen_b ? ex2(fmaf(s[i][2], xb.x, -xb.y)) * xb.z : 0.0f);
                    sum[i][1] += (j + 1 < seen_a ? ex2(fmaf(s[i][1], xa.x, -xa.y)) * xa.z : 0.0f) + (j + 1 < seen_b ? ex2(fmaf(s[i][3], xb.x, -xb.y)) * xb.z : 0.0f);
                }
            }
        }
        if (BUFS == 2) flip ^= 1;
        else __syncthreads();
    }
    float* const mass = a.mass + ((size_t)seq * c.n_kv + h) * c.cap;
    const int old = a.k ? len : end;
#pragma unroll
    for (int i = 0; i < TILES; ++i)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            float x = sum[i][r];
#pragma unroll
            for (int w = 4; w < 32; w <<= 1) x += __shfl_xor_sync(0xffffffffu, x, w);
            if (g == 0) part[warp * (8 * TILES) + 8 * i + 2 * t + r] = x;
        }
    // the ranks' sums, in their order
    cg::cluster_group cluster = cg::this_cluster();
    if (cs > 1) cluster.sync();
    else __syncthreads();
    for (int p = tid; rank == 0 && p < min(S::POS, end - j00); p += 32 * WW) {
        float x = 0.0f;
        for (int r = 0; r < cs; ++r) x += cluster.map_shared_rank(part, r)[p];
        mass[j00 + p] = (j00 + p < old ? mass[j00 + p] : 0.0f) + x;
    }
    if (cs > 1) cluster.sync();                  // no rank leaves while another reads its memory
}

template <int NB>
int launch_prompt_t(const Kv4& c, const Kv4Attend& a, const KvRows& rows, int max_rows, float2* stats, int device, cudaStream_t st) {
    using S = PromptShape<NB>;
    static bool known[64] = {};
    static int resident[64][9];                  // clusters of so many CTAs that the device holds at once
    int here[9], *const room = device < 64 ? resident[device] : here;
    if (device >= 64 || !known[device]) {
        FC_CUDA(cudaFuncSetAttribute(kv4_prompt_kernel<NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM));
        for (int cs = 1; cs <= 8; ++cs) FC_CUDA(resident_clusters((const void*)kv4_prompt_kernel<NB>, dim3(32 * S::WARPS), S::SMEM, cs, &room[cs]));
        if (device < 64) known[device] = true;
    }
    const long long tiles = ((long long)max_rows * a.group + S::COLS - 1) / S::COLS, ctas = tiles * c.n_kv * c.n_seq;
    if (tiles * 8 * c.n_kv > INT_MAX) return fail(FC_E_SHAPE, "%d rows of %d heads are too many for one call", max_rows, c.n_kv * a.group);
    // a cluster shares the positions, two tiles of them each at least, where that shortens the rounds of CTAs; another CTA costs about two tiles (96
    // rows of 32 / 8 heads of 128 behind 30000 positions: 6 CTAs 400 us, 4 492; 600 behind 8000, 152 tiles of columns: 704, unshared 1045).
    // Not beyond two rounds: tiles of a prompt from its start on grow, the largest go first and the rest fill the end (2048 rows of heads of 64: 251, shared 290)
    auto cost = [&](int x) { return (ctas + room[x] - 1) / room[x] * 840 / x * ((c.cap + KT - 1) / KT + 2 * x); };
    int cs = 1;
    for (int x = 2; x <= 8 && ctas <= 2 * room[1]; ++x)
        if (room[x] && x * 2 * KT <= c.cap && cost(x) < cost(cs)) cs = x;
    FC_CUDA(launch_pdl_cluster(kv4_prompt_kernel<NB>, dim3((unsigned)(tiles * cs * c.n_kv), 1, c.n_seq), dim3(32 * S::WARPS), S::SMEM, cs, st, c, a, rows, cs, stats));
    FC_LAUNCHED();
    return FC_OK;
}
template <int NB>
int launch_weights_t(const Kv4& c, const Kv4Attend& a, const KvRows& rows, int max_rows, const float2* stats, int device, cudaStream_t st) {
    using S = WeightsShape<NB>;
    static bool attr_set[64] = {};
    if (device >= 64 || !attr_set[device]) {
        FC_CUDA(cudaFuncSetAttribute(kv4_weights_kernel<NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM));
        if (device < 64) attr_set[device] = true;
    }
    const long long tiles = (c.cap + S::POS - 1) / S::POS, ctas = tiles * c.n_kv * c.n_seq, passes = ((long long)max_rows * a.group + WCOLS - 1) / WCOLS;
    // the first positions are seen by all columns, the last by few: a cluster shares the columns, several rounds of CTAs even out the rest. What the
    // cache holds is on the device: CTAs are counted for its capacity, and 2048 rows in one of 32768 (16 of 17 CTAs leave at once, clusters of 1)
    // take 450 us for their weights where one of 2048 takes 98
    int cs = 1;
    while (cs < 8 && cs * 4 <= passes && ctas * cs < 148 * 8) cs *= 2;
    FC_CUDA(launch_pdl_cluster(kv4_weights_kernel<NB>, dim3((unsigned)(tiles * cs * c.n_kv), 1, c.n_seq), dim3(32 * WW), S::SMEM, cs, st, c, a, rows, cs, stats));
    FC_LAUNCHED();
    return FC_OK;
}

}  // namespace

int launch_kv4_prompt(const Kv4& c, const Kv4Attend& a, const KvRows& rows, int max_rows, float2* stats, int device, cudaStream_t st) {
    switch (c.nb) {
        case 1: return launch_prompt_t<1>(c, a, rows, max_rows, stats, device, st);
        case 2: return launch_prompt_t<2>(c, a, rows, max_rows, stats, device, st);
        case 3: return launch_prompt_t<3>(c, a, rows, max_rows, stats, device, st);
        case 4: return launch_prompt_t<4>(c, a, rows, max_rows, stats, device, st);
        case 5: return launch_prompt_t<5>(c, a, rows, max_rows, stats, device, st);
        case 6: return launch_prompt_t<6>(c, a, rows, max_rows, stats, device, st);
        case 7: return launch_prompt_t<7>(c, a, rows, max_rows, stats, device, st);
        default: return launch_prompt_t<8>(c, a, rows, max_rows, stats, device, st);
    }
}
int launch_kv4_weights(const Kv4& c, const Kv4Attend& a, const KvRows& rows, int max_rows, const float2* stats, int device, cudaStream_t st) {
    switch (c.nb) {
        case 1: return launch_weights_t<1>(c, a, rows, max_rows, stats, device, st);
        case 2: return launch_weights_t<2>(c, a, rows, max_rows, stats, device, st);
        case 3: return launch_weights_t<3>(c, a, rows, max_rows, stats, device, st);
        case 4: return launch_weights_t<4>(c, a, rows, max_rows, stats, device, st);
        case 5: return launch_weights_t<5>(c, a, rows, max_rows, stats, device, st);
        case 6: return launch_weights_t<6>(c, a, rows, max_rows, stats, device, st);
        case 7: return launch_weights_t<7>(c, a, rows, max_rows, stats, device, st);
        default: return launch_weights_t<8>(c, a, rows, max_rows, stats, device, st);
    }
}

}  // namespace fc
