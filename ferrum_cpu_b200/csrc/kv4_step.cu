// Attention of few query rows over the cache of 4-bit levels (layout: kv4.cuh): decode steps and short drafts.
//
// The query rows of a key / value head (rows x heads that share it) are the eight columns of matrix products whose other operand is the
// cache: S^T = K q^T and O^T = V P^T, with levels as they are, exact in f16, and q and P in two f16 planes (22 bits). Up to four
// columns, both planes lie side by side in one product (SPLIT), whose halves are added afterwards: half the products, and half the
// weights a lane has to see to. Keys: a block's sum times its scale is added in f32. (Nibbles as f16 subnormals, with -8 times the sum
// of q to start from, save four instructions a word and cost a digit: 1.8e-6 instead of 2e-7 of the result.) Values: the weight times the
// value's scale is formed in f16 pairs, rn(ph d) and (ph d - rn(ph d)) + pl d of p = ph + pl. Every sum of products of a tile starts anew and
// is added to the row's sums in f32, because the tensor core truncates: what it loses in 32 positions stays below a rounding of the whole.
//
// A cluster shares a (sequence, head): its warps take tiles of 32 positions in turn, each with a running maximum and sum of its
// own and its next tiles on the way to shared memory, and join through distributed shared memory at the end: no scratch memory, nothing
// that two calls could share, one launch. New rows go into the cache on the way, by the CTA whose tile they fall into.
//
// Bound: issue. A tile of heads of 128 is 960 instructions for 4.6 KB, a third of them to form f16 levels: eight sequences of 32767
// positions, 32 query heads on 8, take 102 us, 3.0 TB/s (47 us at the memory's rate; 141 us with the planes in products of their
// own). 64 streams of 255 to 2040 positions, heads of 64, with weights: 40 us. 8 sequences of 8000, 32 (64) query heads on 8: heads of 64 21 us (23), 96
// 26 (29), 128 32 (41), 192 45 (49), 256 53 (65), half as much again with weights. Five to eight columns of heads of 128 spill 380 bytes at the 128 registers
// of two CTAs an SM, those of 256 52 bytes.
#include <cooperative_groups.h>

#include "kv4_frag.cuh"

namespace fc {

namespace {

namespace cg = cooperative_groups;

constexpr int SW = 8, COLS = 8, TILE = 32;        // warps, columns of a product, positions a tile
constexpr int kStepRows = 32;                     // most new rows of a sequence

template <int NB>
struct StepShape {
    static constexpr int DIM = NB * kKvBlock, PAD = DIM + 4;
    static constexpr int STAGES = NB <= 2 ? 3 : 2;
    static constexpr int KBYTES = TILE * NB * 16, DBYTES = TILE * NB * 2, BYTES = 2 * (KBYTES + DBYTES);   // a tile
    static constexpr int RING = SW * STAGES * BYTES;
    static constexpr int FRESH = kStepRows * NB * 36;    // new rows, quantised; then the CTA's joined result
    static constexpr int SMEM = RING + (FRESH > COLS * PAD * 4 ? FRESH : COLS * PAD * 4);
    static constexpr int CTAS = NB <= 4 ? 2 : 1;
};

template <int NB>
__device__ __forceinline__ void ask(const Kv4& c, size_t row, char* tile, int lane, bool values) {
    using S = StepShape<NB>;
    const char *kq = (const char*)(c.kq + row * (NB * 4)), *vq = (const char*)(c.vq + row * (NB * 4));
#pragma unroll
    for (int i = 0; i < NB; ++i) cp16(tile + i * 512 + lane * 16, kq + i * 512 + lane * 16);
    if (values)
#pragma unroll
        for (int i = 0; i < NB; ++i) cp16(tile + S::KBYTES + i * 512 + lane * 16, vq + i * 512 + lane * 16);
    if (lane < 4 * NB) {
        cp16(tile + 2 * S::KBYTES + lane * 16, (const char*)(c.kd + row * NB) + lane * 16);
        if (values) cp16(tile + 2 * S::KBYTES + S::DBYTES + lane * 16, (const char*)(c.vd + row * NB) + lane * 16);
    }
}

// What a lane (g, t) has of q: fragments of channels 32 b + 8 t .. + 7 of its column.
template <int NB, bool SPLIT>
struct Query {
    uint32_t f[NB][4];                           // SPLIT: of plane g / 4 of column g % 4; else the high plane of column g
    uint32_t r[SPLIT ? 1 : NB][4];               // the low plane
    float inv0, inv1;                            // of this lane's columns of scores
};

// The scores of a tile. SPLIT: s[m][0..1] are position 16 m + g + 8 (t / 2), columns 2 (t % 2) and + 1. Else s[m][0..1] position 16 m + g,
// columns 2 t and + 1, s[m][2..3] position 16 m + g + 8. With `edge`, -inf behind what a column sees.
template <int NB, bool SPLIT>
__device__ __forceinline__ void tile_scores(const char* tile, const Query<NB, SPLIT>& q, bool edge, int j0, int seen0, int seen1, int g, int t, float (&s)[2][SPLIT ? 2 : 4]) {
    using S = StepShape<NB>;
    const uint32_t* kq = (const uint32_t*)tile;
    const __half* kd = (const __half*)(tile + 2 * S::KBYTES);
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        uint32_t w0[NB], w1[NB];
        float d0[NB], d1[NB], x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        const int r = 16 * m + g;
        load_words(kq + r * (NB * 4) + t * NB, w0);
        load_words(kq + (r + 8) * (NB * 4) + t * NB, w1);
        load_scales(kd + r * NB, d0);
        load_scales(kd + (r + 8) * NB, d1);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            uint32_t f0[4], f1[4];
            levels_of(w0[b], f0);
            levels_of(w1[b], f1);
            const uint32_t a0[4] = {f0[0], f1[0], f0[1], f1[1]}, a1[4] = {f0[2], f1[2], f0[3], f1[3]};
            float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            mma16816(y, a0, q.f[b][0], q.f[b][1]);
            mma16816(y, a1, q.f[b][2], q.f[b][3]);
            if (!SPLIT) {
                constexpr int ONE = SPLIT ? 0 : 1;
                float z[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                mma16816(z, a0, q.r[b * ONE][0], q.r[b * ONE][1]);
                mma16816(z, a1, q.r[b * ONE][2], q.r[b * ONE][3]);
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] += z[e];
            }
            x[0] = fmaf(y[0], d0[b], x[0]);
            x[1] = fmaf(y[1], d0[b], x[1]);
            x[2] = fmaf(y[2], d1[b], x[2]);
            x[3] = fmaf(y[3], d1[b], x[3]);
        }
        if (SPLIT) {
            // the planes of a column meet: lanes t < 2 keep position g, the others position g + 8
            const bool upper = t >= 2;
            const float y0 = __shfl_xor_sync(0xffffffffu, upper ? x[0] : x[2], 2), y1 = __shfl_xor_sync(0xffffffffu, upper ? x[1] : x[3], 2);
            s[m][0] = ((upper ? x[2] : x[0]) + y0) * q.inv0;
            s[m][1] = ((upper ? x[3] : x[1]) + y1) * q.inv1;
            if (edge) {
                const int j = j0 + r + 8 * (t >> 1);
                s[m][0] = j < seen0 ? s[m][0] : -INFINITY;
                s[m][1] = j < seen1 ? s[m][1] : -INFINITY;
            }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[m][SPLIT ? 0 : e] = x[e] * (e & 1 ? q.inv1 : q.inv0);
                if (edge) s[m][SPLIT ? 0 : e] = j0 + r + 8 * (e >> 1) < (e & 1 ? seen1 : seen0) ? s[m][SPLIT ? 0 : e] : -INFINITY;
            }
        }
    }
}

__device__ __forceinline__ uint32_t hmaxabs2u(uint32_t a, uint32_t b) {
    const __half2 r = __hmax2(*(const __half2*)&a, __habs2(*(const __half2*)&b));
    return *(const uint32_t*)&r;
}

// The n-th longest sequence (the first of equals first). All threads of the CTA; s: n_seq + 1 words, free again behind the call.
__device__ __forceinline__ int nth_longest(const int* __restrict__ lens, int n_seq, int n, int* s) {
    const int tid = threadIdx.x;
    static_assert(32 * SW >= kKvMaxSeq, "a thread for each sequence");
    const int mine = tid < n_seq ? lens[tid] : 0;
    if (tid < n_seq) s[tid] = mine;
    __syncthreads();
    if (tid < n_seq) {
        int before = 0;
        for (int q = 0; q < n_seq; ++q) before += s[q] > mine || (s[q] == mine && q < tid);
        if (before == n) s[n_seq] = tid;
    }
    __syncthreads();
    const int seq = s[n_seq];
    __syncthreads();
    return seq;
}

template <int NB, bool SPLIT>
__global__ void __launch_bounds__(32 * SW, StepShape<NB>::CTAS) kv4_step_kernel(Kv4 c, Kv4Attend a, KvRows rows, int by_length, float2* __restrict__ stats) {
    using S = StepShape<NB>;
    constexpr int DIM = S::DIM, PAD = S::PAD, CALL = SPLIT ? COLS / 2 : COLS;      // columns of a call
    extern __shared__ __align__(16) char smem[];
    __shared__ float2 warp_ml[SW][COLS];          // running maximum (base 2) and sum
    __shared__ float warp_f[SW][COLS];
    __shared__ float2 cta_ml[COLS];
    pdl_trigger();
    pdl_wait();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int cs = gridDim.x, rank = blockIdx.x, h = blockIdx.y % c.n_kv, col0 = blockIdx.y / c.n_kv * CALL;
    const int seq = by_length ? nth_longest(a.lens, c.n_seq, blockIdx.z, (int*)smem) : blockIdx.z;
    const int first = rows.start[seq], n = rows.start[seq + 1] - first, cols = min(n * a.group - col0, CALL);
    if (cols <= 0) return;                        // the whole cluster
    const int len = a.lens[seq], end = a.k ? len + n : len;
    float* const out = a.out + (size_t)first * a.ldo + (size_t)h * a.group * DIM;
    auto place = [&](int col) { const int i = (col0 + col) / a.group; return (size_t)i * a.ldo + ((col0 + col) - i * a.group) * DIM; };
    if (len < 0 || len > c.cap - (a.k ? n : 0)) {
        for (int e = rank * (32 * SW) + tid; e < cols * DIM; e += cs * (32 * SW)) out[place(e / DIM) + e % DIM] = __int_as_float(0x7fffffff);
        return;
    }
    const int base = end - n + 1;                 // row i sees the positions below base + i
    const int tiles = (max(0, base + (col0 + cols - 1) / a.group) + TILE - 1) / TILE, stride = cs * SW, mine = rank * SW + warp;
    const size_t row0 = c.row(seq, h, 0);
    char* const ring = smem + warp * (S::STAGES * S::BYTES);
    char* const fresh = smem + S::RING;
#pragma unroll
    for (int i = 0; i < S::STAGES - 1; ++i) {
        if (mine + i * stride < tiles) ask<NB>(c, row0 + (size_t)(mine + i * stride) * TILE, ring + i * S::BYTES, lane, true);
        cp_commit();
    }

    // the CTA's share of the new rows: words of keys, half words of values, scales, as a tile has them
    const int new0 = a.k ? len / TILE : tiles;
    bool any = false;
    for (int tile = new0; tile < tiles; ++tile) any |= tile % stride / SW == rank;
    if (any) {
        constexpr int PARTS = (NB + 3) / 4;
        for (int w = warp; w < n * PARTS * 2; w += SW) {
            const int i = w / (PARTS * 2), pos = len + i, tile = pos / TILE, b = w / 2 % PARTS * 4 + (lane >> 3), e = lane & 7;
            if (tile >= tiles || tile % stride / SW != rank) continue;
            const float* x = w & 1 ? a.v : a.k;
            const bool in = b < NB;
            const float4 v = in ? *(const float4*)(x + (size_t)(first + i) * a.ldkv + h * DIM + b * kKvBlock + 4 * e) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            __half d;
            int level[4];
            quantize4(v, &d, level);
            const size_t row = row0 + pos;
            if (w & 1) {
                const uint2 half = value_halves(level, lane);
                if (in && e < 2) {
                    uint16_t* to = (uint16_t*)c.vq + 2 * ((row >> 1) * (NB * 8) + (4 * e) * NB + b) + (pos & 1);
                    uint16_t* keep = (uint16_t*)(fresh + i * (NB * 36) + NB * 16) + (4 * e) * NB + b;
                    to[0] = keep[0] = (uint16_t)half.x; to[2 * NB] = keep[NB] = (uint16_t)(half.x >> 16);
                    to[4 * NB] = keep[2 * NB] = (uint16_t)half.y; to[6 * NB] = keep[3 * NB] = (uint16_t)(half.y >> 16);
                }
                if (in && !e) { c.vd[row * NB + b] = d; ((__half*)(fresh + i * (NB * 36) + NB * 34))[b] = d; }
            } else {
                const uint32_t word = key_word(level, lane);
                if (in && !(e & 1)) {
                    c.kq[row * (NB * 4) + (e >> 1) * NB + b] = word;
                    ((uint32_t*)(fresh + i * (NB * 36)))[(e >> 1) * NB + b] = word;
                }
                if (in && !e) { c.kd[row * NB + b] = d; ((__half*)(fresh + i * (NB * 36) + NB * 32))[b] = d; }
            }
        }
        __syncthreads();
    }

    // q: brought to [2^13, 2^14) by a power of two a column
    const int col = SPLIT ? g & 3 : g, plane = SPLIT ? g >> 2 : 0;
    const uint32_t minus = plane ? 0xbc00bc00u : 0u;      // what the high plane of a weight's product is taken times in this lane
    const int c0 = SPLIT ? 2 * (t & 1) : 2 * t, c1 = c0 + 1;          // this lane's columns of scores
    Query<NB, SPLIT> q;
    {
        float x[NB][8];
        const bool live = col < cols;
        const int i = (col0 + col) / a.group, head = h * a.group + (col0 + col) - i * a.group;
        const float* from = a.q + (size_t)(first + i) * a.ldq + (size_t)head * DIM + 8 * t;
        const float scale = a.scale * 1.44269504f;
        float top = 0.0f;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const float4 lo = live ? *(const float4*)(from + 32 * b) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            const float4 hi = live ? *(const float4*)(from + 32 * b + 4) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            const float v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
            for (int j = 0; j < 8; ++j) { x[b][j] = v[j] * scale; top = fmaxf(top, fabsf(x[b][j])); }
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int shift = plane_shift(top);
        const float up = exp2i(shift), inv = exp2i(-shift);
        q.inv0 = __shfl_sync(0xffffffffu, inv, 4 * c0);
        q.inv1 = __shfl_sync(0xffffffffu, inv, 4 * c1);
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t hi, lo;
                planes_of(x[b][j] * up, x[b][j + 4] * up, &hi, &lo);
                q.f[b][j] = SPLIT && plane ? lo : hi;
                if (!SPLIT) q.r[SPLIT ? 0 : b][j] = lo;
            }
    }
    auto sees = [&](int x) { return x < cols ? base + (col0 + x) / a.group : 0; };
    const int seen0 = sees(c0), seen1 = sees(c1), seen_g = sees(col);
    const int whole_tiles = cols == CALL ? max(0, base + col0 / a.group) / TILE : 0;      // that every column sees whole

    float o[NB][2][4] = {}, m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;
    float s[2][SPLIT ? 2 : 4];
    int stage = 0;
    for (int tile = mine; tile < tiles; tile += stride) {
        char* at = ring + stage * S::BYTES;
        {
            const int ahead = tile + (S::STAGES - 1) * stride;
            const int to = stage == 0 ? S::STAGES - 1 : stage - 1;
            __syncwarp();                         // its readers are done
            if (ahead < tiles) ask<NB>(c, row0 + (size_t)ahead * TILE, ring + to * S::BYTES, lane, true);
            cp_commit();
        }
        cp_wait<S::STAGES - 1>();
        __syncwarp();
        const int j0 = tile * TILE;
        const bool edge = tile >= whole_tiles;
        if (a.k && j0 + TILE > len) {
            // new rows over what the tile holds of them
            for (int r = max(len - j0, 0); r < TILE && j0 + r < len + n; ++r) {
                const char* from = fresh + (j0 + r - len) * (NB * 36);
                if (lane < 4 * NB) ((uint32_t*)at)[r * (NB * 4) + lane] = ((const uint32_t*)from)[lane];
                for (int e = lane; e < 8 * NB; e += 32)
                    ((uint16_t*)(at + S::KBYTES))[2 * ((r >> 1) * (NB * 8) + e) + (r & 1)] = ((const uint16_t*)(from + NB * 16))[e];
                if (lane < NB) {
                    ((__half*)(at + 2 * S::KBYTES))[r * NB + lane] = ((const __half*)(from + NB * 32))[lane];
                    ((__half*)(at + 2 * S::KBYTES + S::DBYTES))[r * NB + lane] = ((const __half*)(from + NB * 34))[lane];
                }
            }
            __syncwarp();
        }
        tile_scores<NB, SPLIT>(at, q, edge, j0, seen0, seen1, g, t, s);
        float t0 = fmaxf(s[0][0], s[1][0]), t1 = fmaxf(s[0][1], s[1][1]);
        if (!SPLIT) {
            constexpr int LO = SPLIT ? 0 : 2, HI = SPLIT ? 1 : 3;
            t0 = fmaxf(t0, fmaxf(s[0][LO], s[1][LO]));
            t1 = fmaxf(t1, fmaxf(s[0][HI], s[1][HI]));
        }
#pragma unroll
        for (int w = SPLIT ? 2 : 4; w < 32; w <<= 1) {
            t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, w));
            t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, w));
        }
        t0 = fmaxf(t0, m0);
        t1 = fmaxf(t1, m1);
        const float z0 = (t0 == -INFINITY ? 0.0f : t0) - kLift, z1 = (t1 == -INFINITY ? 0.0f : t1) - kLift;
        if (__any_sync(0xffffffffu, t0 != m0 || t1 != m1)) {
            const float f0 = ex2(m0 - kLift - z0), f1 = ex2(m1 - kLift - z1);
            l0 *= f0; l1 *= f1;
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int u = 0; u < 2; ++u) { o[b][u][0] *= f0; o[b][u][1] *= f1; o[b][u][2] *= f0; o[b][u][3] *= f1; }
            m0 = t0; m1 = t1;
        }
        // weights as planes, from (position, columns) to (positions 2 t, 2 t + 1 and 2 t + 8, 2 t + 9, column g)
        uint32_t ph[2][2], pl[2][2];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            if (SPLIT) {
                const float x = ex2(s[m][0] - z0), y = ex2(s[m][1] - z1);
                l0 += x; l1 += y;
                const uint32_t xb = __float_as_uint(x), yb = __float_as_uint(y);
                const uint32_t hi = movmatrix(__byte_perm(xb, yb, 0x7632)), lo = movmatrix(__byte_perm(xb, yb, 0x5410));
                // lanes g < 4 have positions 2 t, 2 t + 1 of column g, the others 2 t + 8, 2 t + 9 of column g - 4
                uint32_t h0, r0;
                planes_of(__uint_as_float(__byte_perm(lo, hi, 0x5410)), __uint_as_float(__byte_perm(lo, hi, 0x7632)), &h0, &r0);
                const uint32_t h1 = __shfl_xor_sync(0xffffffffu, h0, 16), r1 = __shfl_xor_sync(0xffffffffu, r0, 16);
                ph[m][0] = plane ? h1 : h0; ph[m][1] = plane ? h0 : h1;
                pl[m][0] = plane ? r1 : 0u; pl[m][1] = plane ? r0 : 0u;
            } else {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const float x = ex2(s[m][SPLIT ? 0 : 2 * u] - z0), y = ex2(s[m][SPLIT ? 1 : 2 * u + 1] - z1);
                    l0 += x; l1 += y;
                    const uint32_t xb = __float_as_uint(x), yb = __float_as_uint(y);
                    const uint32_t hi = movmatrix(__byte_perm(xb, yb, 0x7632)), lo = movmatrix(__byte_perm(xb, yb, 0x5410));
                    planes_of(__uint_as_float(__byte_perm(lo, hi, 0x5410)), __uint_as_float(__byte_perm(lo, hi, 0x7632)), &ph[m][u], &pl[m][u]);
                }
            }
        }
        // scales of the values in pairs of positions, times a power of two that brings the largest of the tile to 2^kScaleLift and above
        // (2^15 at most): the largest that column g sees, as what lies behind must not change a bit
        const __half* vd = (const __half*)(at + 2 * S::KBYTES + S::DBYTES);
        uint32_t d[2][2][NB], most = 0;
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                uint32_t w[NB];                   // the scales of two positions, one after the other
                load_words((const uint32_t*)(vd + (16 * m + 2 * t + 8 * u) * NB), w);
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const int x = b, y = NB + b;  // halves of w
                    d[m][u][b] = __byte_perm(w[x >> 1], w[y >> 1], (x & 1 ? 0x32 : 0x10) | (y & 1 ? 0x7600 : 0x5400));
                }
                if (edge) {                       // what a weight of 0 meets is 0: what lies there could be large
                    const int j = j0 + 16 * m + 2 * t + 8 * u;
                    const uint32_t sight = (j < seen_g ? 0xffffu : 0u) | (j + 1 < seen_g ? 0xffff0000u : 0u);
#pragma unroll
                    for (int b = 0; b < NB; ++b) d[m][u][b] &= sight;
                }
#pragma unroll
                for (int b = 0; b < NB; ++b) most = hmaxabs2u(most, d[m][u][b]);
            }
        most = hmaxabs2u(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = hmaxabs2u(most, __shfl_xor_sync(0xffffffffu, most, 2));
        const int exponent = (int)(max(most & 0xffffu, most >> 16) >> 10), lift = min(15 + kScaleLift - exponent, 15);
        const uint32_t by = (uint32_t)(15 + lift) << 10;      // 2^lift, -8 <= lift
        const uint32_t up = by | by << 16;
        const float down = exp2i(-lift), down0 = edge ? __shfl_sync(0xffffffffu, down, 4 * c0) : down, down1 = edge ? __shfl_sync(0xffffffffu, down, 4 * c1) : down;
        const uint32_t* vq = (const uint32_t*)(at + S::KBYTES);
        uint32_t w[4][NB];                        // pairs of positions t, t + 4, t + 8, t + 12
#pragma unroll
        for (int u = 0; u < 4; ++u) load_words(vq + (t + 4 * u) * (NB * 8) + g * NB, w[u]);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            float x[2][4] = {};
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                uint32_t hi[2], lo[2], e0[4], e1[4];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const uint32_t f = hmul2u(d[m][u][b], up);
                    hi[u] = hmul2u(ph[m][u], f);
                    if (SPLIT) {
                        // the low plane's lanes: minus the high plane, and the rest of the weight (kept for them alone)
                        hi[u] = hfma2u(pl[m][u], f, hfma2u(ph[m][u], f, hmul2u(hi[u], minus)));
                    } else {
                        lo[u] = hfma2u(pl[m][u], f, hfms2u(ph[m][u], f, hi[u]));
                    }
                }
                levels_of(w[2 * m][b], e0);
                levels_of(w[2 * m + 1][b], e1);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const uint32_t f[4] = {e0[2 * u], e0[2 * u + 1], e1[2 * u], e1[2 * u + 1]};
                    if (!SPLIT) mma16816(x[u], f, lo[0], lo[1]);
                    mma16816(x[u], f, hi[0], hi[1]);
                }
            }
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[b][u][e] = fmaf(x[u][e], e & 1 ? down1 : down0, o[b][u][e]);
        }
        stage = stage + 1 == S::STAGES ? 0 : stage + 1;
    }
    cp_wait<0>();
    __syncwarp();
#pragma unroll
    for (int w = SPLIT ? 2 : 4; w < 32; w <<= 1) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, w);
        l1 += __shfl_xor_sync(0xffffffffu, l1, w);
    }
    if (g == 0 && (!SPLIT || t < 2)) {
        warp_ml[warp][c0] = make_float2(m0, l0);
        warp_ml[warp][c1] = make_float2(m1, l1);
    }
    float* const mo = (float*)ring;               // [column][channel]
    if (SPLIT) {
        // the planes of a weight meet: lanes t < 2 keep channels g, the others channels g + 8
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const bool upper = t >= 2;
                const float y0 = __shfl_xor_sync(0xffffffffu, upper ? o[b][u][0] : o[b][u][2], 2), y1 = __shfl_xor_sync(0xffffffffu, upper ? o[b][u][1] : o[b][u][3], 2);
                const int ch = 32 * b + 16 * u + g + (upper ? 8 : 0);
                mo[c0 * PAD + ch] = (upper ? o[b][u][2] : o[b][u][0]) + y0;
                mo[c1 * PAD + ch] = (upper ? o[b][u][3] : o[b][u][1]) + y1;
            }
    } else {
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int ch = 32 * b + 16 * u + g;
                mo[c0 * PAD + ch] = o[b][u][0];
                mo[c1 * PAD + ch] = o[b][u][1];
                mo[c0 * PAD + ch + 8] = o[b][u][2];
                mo[c1 * PAD + ch + 8] = o[b][u][3];
            }
    }
    __syncthreads();
    if (tid < SW * CALL) {
        const int x = tid % CALL;
        float m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int w = 0; w < SW; ++w) m = fmaxf(m, warp_ml[w][x].x);
        const float z = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int w = 0; w < SW; ++w) l += warp_ml[w][x].y * ex2(warp_ml[w][x].x - z);
        warp_f[tid / CALL][x] = ex2(warp_ml[tid / CALL][x].x - z);
        if (tid < CALL) cta_ml[x] = make_float2(m, l);
    }
    __syncthreads();
    float* const joined = (float*)fresh;          // the new rows in it have been read
    for (int e = tid; e < CALL * DIM; e += 32 * SW) {
        const int x = e / DIM, ch = e % DIM;
        float y = 0.0f;
#pragma unroll
        for (int w = 0; w < SW; ++w) y = fmaf(((const float*)(smem + w * (S::STAGES * S::BYTES)))[x * PAD + ch], warp_f[w][x], y);
        if (cs == 1) {
            if (x < cols) out[place(x) + ch] = cta_ml[x].y == 0.0f ? 0.0f : y / cta_ml[x].y;
        } else {
            joined[x * PAD + ch] = y;
        }
    }
    cg::cluster_group cluster = cg::this_cluster();
    if (cs > 1) cluster.sync();
    // a column's maximum and sum over the ranks
    auto whole = [&](int x, float* z) {
        float m = -INFINITY, l = 0.0f;
        for (int r = 0; r < cs; ++r) m = fmaxf(m, cluster.map_shared_rank(cta_ml, r)[x].x);
        *z = m == -INFINITY ? 0.0f : m;
        for (int r = 0; r < cs; ++r) {
            const float2 y = cluster.map_shared_rank(cta_ml, r)[x];
            l = fmaf(y.y, ex2(y.x - *z), l);
        }
        return l;
    };
    // every rank joins its share of the elements
    for (int e = rank * (32 * SW) + tid; cs > 1 && e < cols * DIM; e += cs * (32 * SW)) {
        const int x = e / DIM, ch = e % DIM;
        float z, y = 0.0f;
        const float l = whole(x, &z);
        for (int r = 0; r < cs; ++r) y = fmaf(cluster.map_shared_rank(joined, r)[x * PAD + ch], ex2(cluster.map_shared_rank(cta_ml, r)[x].x - z), y);
        out[place(x) + ch] = l == 0.0f ? 0.0f : y / l;
    }
    if (stats && rank == 0 && tid < cols) {
        float z;
        const float l = whole(tid, &z);
        stats[((size_t)first + (col0 + tid) / a.group) * (c.n_kv * a.group) + h * a.group + (col0 + tid) % a.group] = make_float2(z - kLift, l);
    }
    if (a.mass && !stats) {
        // the weights once more, against the whole row's maximum and sum: the last tile's scores are still there
        float z0, z1;
        l0 = whole(c0, &z0);
        l1 = whole(c1, &z1);
        l0 = c0 < cols && l0 != 0.0f ? 1.0f / l0 : 0.0f;
        l1 = c1 < cols && l1 != 0.0f ? 1.0f / l1 : 0.0f;
        z0 -= kLift; z1 -= kLift;
        float* const mass = a.mass + ((size_t)seq * c.n_kv + h) * c.cap;
        if (cs > 1) cluster.sync();               // the ring may be written, and no rank leaves while it is read
        else __syncthreads();
        const int last = tiles > mine ? mine + (tiles - 1 - mine) / stride * stride : -1;
#pragma unroll
        for (int i = 1; i < S::STAGES; ++i) {
            if (last - i * stride >= 0) ask<NB>(c, row0 + (size_t)(last - i * stride) * TILE, ring + i * S::BYTES, lane, false);
            cp_commit();
        }
        // what the tile's positions had is asked for a tile ahead
        constexpr int EACH = SPLIT ? 1 : 2;
        const bool mine_to_add = (SPLIT ? t & 1 : t) == 0;
        const int old_end = a.k ? len : end;
        auto spot = [&](int tile, int m, int u) { return tile * TILE + 16 * m + g + 8 * (SPLIT ? t >> 1 : u); };
        float had[2][EACH], next[2][EACH] = {};
        auto ask_mass = [&](int tile, float (&x)[2][EACH]) {
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int u = 0; u < EACH; ++u) {
                    const int j = spot(tile, m, u);
                    x[m][u] = mine_to_add && tile >= 0 && j < old_end ? mass[j] : 0.0f;
                }
        };
        ask_mass(last, next);
        stage = 0;
        for (int tile = last; tile >= 0; tile -= stride) {
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int u = 0; u < EACH; ++u) had[m][u] = next[m][u];
            ask_mass(tile - stride, next);
            if (tile != last) {
                cp_wait<S::STAGES - 2>();
                __syncwarp();
                tile_scores<NB, SPLIT>(ring + stage * S::BYTES, q, true, tile * TILE, seen0, seen1, g, t, s);
                __syncwarp();
            }
            if (tile - S::STAGES * stride >= 0) ask<NB>(c, row0 + (size_t)(tile - S::STAGES * stride) * TILE, ring + stage * S::BYTES, lane, false);
            cp_commit();
            stage = stage + 1 == S::STAGES ? 0 : stage + 1;
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int u = 0; u < EACH; ++u) {
                    float x = (l0 != 0.0f ? ex2(s[m][2 * u] - z0) * l0 : 0.0f) + (l1 != 0.0f ? ex2(s[m][2 * u + 1] - z1) * l1 : 0.0f);
                    x += __shfl_xor_sync(0xffffffffu, x, 1);
                    if (!SPLIT) x += __shfl_xor_sync(0xffffffffu, x, 2);
                    const int j = spot(tile, m, u);
                    if (mine_to_add && j < end) mass[j] = had[m][u] + x;
                }
        }
        return;
    }
    if (cs > 1) cluster.sync();                   // no rank leaves while another reads its memory
}

template <int NB, bool SPLIT>
int launch_step_t(const Kv4& c, const Kv4Attend& a, const KvRows& rows, int groups, float2* stats, int device, cudaStream_t st) {
    using S = StepShape<NB>;
    const auto kernel = kv4_step_kernel<NB, SPLIT>;
    static bool known[64] = {};
    static int resident[64][9];                   // clusters of so many CTAs that the device holds at once
    int here[9], *const room = device < 64 ? resident[device] : here;
    if (device >= 64 || !known[device]) {
        FC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM));
        for (int cs = 1; cs <= 8; ++cs) FC_CUDA(resident_clusters((const void*)kernel, dim3(32 * SW), S::SMEM, cs, &room[cs]));
        if (device < 64) known[device] = true;
    }
    // as many CTAs for a sequence's head as are resident together, as long as each takes tiles off the warps' shares. What is resident is asked for,
    // not computed: clusters of 5 or 7 leave SMs of a processing cluster unused. 80 heads of 8000 positions: 3 CTAs, 40 us (2: 54), 40 heads of
    // 32000: 6, 70 us (4: 98; 7, in two waves: 90), of 2000: 4, 10.4 us (6, with as many tiles a warp: 11.2)
    const long long clusters = (long long)c.n_seq * c.n_kv * groups;
    const int tiles = (c.cap + TILE - 1) / TILE;
    auto share = [&](int x) { return (tiles + SW * x - 1) / (SW * x); };
    int cs = 1;
    for (int x = 2; x <= 8; ++x)
        if (clusters <= room[x] && share(x) < share(cs)) cs = x;
    // more CTAs than are resident: the long sequences go first (64 streams of 255 to 2040 positions, weights kept: 40 us, in
    // the order of the call 47)
    const int by_length = clusters > room[cs] && c.n_seq > 1;
    FC_CUDA(launch_pdl_cluster(kernel, dim3(cs, c.n_kv * groups, c.n_seq), dim3(32 * SW), S::SMEM, cs, st, c, a, rows, by_length, stats));
    FC_LAUNCHED();
    return FC_OK;
}

template <int NB>
int launch_step_nb(const Kv4& c, const Kv4Attend& a, const KvRows& rows, int cols, float2* stats, int device, cudaStream_t st) {
    const bool split = cols <= COLS / 2;
    const int groups = split ? 1 : (cols + COLS - 1) / COLS;
    return split ? launch_step_t<NB, true>(c, a, rows, groups, stats, device, st) : launch_step_t<NB, false>(c, a, rows, groups, stats, device, st);
}

}  // namespace

bool kv4_step_covers(const Kv4& c, int group, int max_rows) {
    // Every group of 8 columns reads the cache anew, the prompt kernel reads it once for 128. Step / prompt, us, heads on 8 (1 the last):
    //   columns                         16         32         64
    //   1 x 900 positions of 64      9.2 / 12.1  10.1 / 12.4  13.4 / 13.1
    //   1 x 30000 of 64               36 / 84     38 / 86     67 / 91
    //   16 x 2000 of 64               22 / 48     44 / 50     76 / 53
    //   8 x 8000 of 128               71 / 204   125 / 209   240 / 220
    //   1 x 30000 of 128, 1 head      42 / 180    43 / 182    48 / 189
    // Only full devices lose, at 64. Groups of columns and heads lie on the grid's y.
    const long long cols = (long long)max_rows * group;
    return max_rows <= kStepRows && cols <= 64 && c.n_kv * ((cols + COLS - 1) / COLS) <= 65535;
}

int launch_kv4_step(const Kv4& c, const Kv4Attend& a, const KvRows& rows, int max_rows, float2* stats, int device, cudaStream_t st) {
    const int cols = max_rows * a.group;
    switch (c.nb) {
        case 1: return launch_step_nb<1>(c, a, rows, cols, stats, device, st);
        case 2: return launch_step_nb<2>(c, a, rows, cols, stats, device, st);
        case 3: return launch_step_nb<3>(c, a, rows, cols, stats, device, st);
        case 4: return launch_step_nb<4>(c, a, rows, cols, stats, device, st);
        case 5: return launch_step_nb<5>(c, a, rows, cols, stats, device, st);
        case 6: return launch_step_nb<6>(c, a, rows, cols, stats, device, st);
        case 7: return launch_step_nb<7>(c, a, rows, cols, stats, device, st);
        default: return launch_step_nb<8>(c, a, rows, cols, stats, device, st);
    }
}

}  // namespace fc
