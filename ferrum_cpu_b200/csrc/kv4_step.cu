// Attention of few query rows over the cache of 4-bit levels (layout: kv4.cuh): decode steps and short drafts.
//
// The query rows of a key / value head (rows x heads that share it) are the eight columns of matrix products whose other operand is the
// cache: S^T = K q^T with levels as they are (exact in f16) and q in two f16 planes, a block's sum times its f16 scale in f32;
// O^T = V P^T with the weights times the value's scale in two planes. Every sum of products of a tile starts from zero and is added to the
// row's sums in f32, because the tensor core truncates: what it loses in a tile of 32 positions stays below a rounding of the whole.
//
// A cluster shares a (sequence, head): its warps take tiles of 32 positions in turn, each with a running maximum and sum of its
// own and its next tiles on the way to shared memory, and join through distributed shared memory at the end: no scratch memory, nothing
// that two calls could share, one launch. New rows go into the cache on the way, by the CTA whose tile they fall into.
#include <cooperative_groups.h>

#include "kv4_frag.cuh"

namespace fc {

namespace {

namespace cg = cooperative_groups;

constexpr int SW = 8, COLS = 8, TILE = 32;
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

// The scores of a tile: s[m][0..1]: position 16 m + g, columns 2 t and 2 t + 1; s[m][2..3]: position 16 m + g + 8. -inf behind what a column sees.
template <int NB>
__device__ __forceinline__ void tile_scores(const char* tile, const uint32_t (&qh)[NB][4], const uint32_t (&ql)[NB][4], float inv0, float inv1, int j0, int seen0,
                                            int seen1, int g, int t, float (&s)[2][4]) {
    using S = StepShape<NB>;
    const uint32_t* kq = (const uint32_t*)tile;
    const __half* kd = (const __half*)(tile + 2 * S::KBYTES);
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        uint32_t w0[NB], w1[NB];
        float d0[NB], d1[NB];
        const int r = 16 * m + g;
        load_words(kq + r * (NB * 4) + t * NB, w0);
        load_words(kq + (r + 8) * (NB * 4) + t * NB, w1);
        load_scales(kd + r * NB, d0);
        load_scales(kd + (r + 8) * NB, d1);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[m][i] = 0.0f;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            uint32_t f0[4], f1[4];
            levels_of(w0[b], f0);
            levels_of(w1[b], f1);
            const uint32_t a0[4] = {f0[0], f1[0], f0[1], f1[1]}, a1[4] = {f0[2], f1[2], f0[3], f1[3]};
            float x[4] = {0.0f, 0.0f, 0.0f, 0.0f}, y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            mma16816(x, a0, qh[b][0], qh[b][1]);
            mma16816(y, a0, ql[b][0], ql[b][1]);
            mma16816(x, a1, qh[b][2], qh[b][3]);
            mma16816(y, a1, ql[b][2], ql[b][3]);
            s[m][0] = fmaf(x[0] + y[0], d0[b], s[m][0]);
            s[m][1] = fmaf(x[1] + y[1], d0[b], s[m][1]);
            s[m][2] = fmaf(x[2] + y[2], d1[b], s[m][2]);
            s[m][3] = fmaf(x[3] + y[3], d1[b], s[m][3]);
        }
        s[m][0] = j0 + r < seen0 ? s[m][0] * inv0 : -INFINITY;
        s[m][1] = j0 + r < seen1 ? s[m][1] * inv1 : -INFINITY;
        s[m][2] = j0 + r + 8 < seen0 ? s[m][2] * inv0 : -INFINITY;
        s[m][3] = j0 + r + 8 < seen1 ? s[m][3] * inv1 : -INFINITY;
    }
}

template <int NB>
__global__ void __launch_bounds__(32 * SW, StepShape<NB>::CTAS) kv4_step_kernel(Kv4 c, Kv4Attend a, KvRows rows, float2* __restrict__ stats) {
    using S = StepShape<NB>;
    constexpr int DIM = S::DIM, PAD = S::PAD;
    extern __shared__ __align__(16) char smem[];
    __shared__ float2 warp_ml[SW][COLS];          // running maximum (base 2) and sum
    __shared__ float warp_f[SW][COLS];
    __shared__ float2 cta_ml[COLS];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int cs = gridDim.x, rank = blockIdx.x, h = blockIdx.y % c.n_kv, col0 = blockIdx.y / c.n_kv * COLS, seq = blockIdx.z;
    const int first = rows.start[seq], n = rows.start[seq + 1] - first, cols = min(n * a.group - col0, COLS);
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

    // column g of this lane's fragments: channels 32 b + 8 t .. + 7 as two planes, brought to [2^13, 2^14) by a power of two
    uint32_t qh[NB][4], ql[NB][4];
    float inv;
    {
        float x[NB][8];
        const bool live = g < cols;
        const int i = (col0 + g) / a.group, head = h * a.group + (col0 + g) - i * a.group;
        const float* q = a.q + (size_t)(first + i) * a.ldq + (size_t)head * DIM + 8 * t;
        const float scale = a.scale * 1.44269504f;
        float top = 0.0f;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const float4 lo = live ? *(const float4*)(q + 32 * b) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            const float4 hi = live ? *(const float4*)(q + 32 * b + 4) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            const float v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
            for (int j = 0; j < 8; ++j) { x[b][j] = v[j] * scale; top = fmaxf(top, fabsf(x[b][j])); }
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int shift = plane_shift(top);
        const float up = exp2i(shift);
        inv = exp2i(-shift);
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int j = 0; j < 4; ++j) planes_of(x[b][j] * up, x[b][j + 4] * up, &qh[b][j], &ql[b][j]);
    }
    const float inv0 = __shfl_sync(0xffffffffu, inv, 8 * t), inv1 = __shfl_sync(0xffffffffu, inv, 8 * t + 4);
    const int seen0 = 2 * t < cols ? base + (col0 + 2 * t) / a.group : 0, seen1 = 2 * t + 1 < cols ? base + (col0 + 2 * t + 1) / a.group : 0;

    const int seen_g = g < cols ? base + (col0 + g) / a.group : 0;

    float o[NB][2][4] = {}, m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;
    float s[2][4];
    int stage = 0;
    for (int tile = mine, i = 0; tile < tiles; tile += stride, ++i) {
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
        tile_scores<NB>(at, qh, ql, inv0, inv1, j0, seen0, seen1, g, t, s);
        float t0 = fmaxf(fmaxf(s[0][0], s[0][2]), fmaxf(s[1][0], s[1][2])), t1 = fmaxf(fmaxf(s[0][1], s[0][3]), fmaxf(s[1][1], s[1][3]));
#pragma unroll
        for (int w = 4; w < 32; w <<= 1) {
            t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, w));
            t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, w));
        }
        t0 = fmaxf(t0, m0);
        t1 = fmaxf(t1, m1);
        const float z0 = t0 == -INFINITY ? 0.0f : t0, z1 = t1 == -INFINITY ? 0.0f : t1;
        if (__any_sync(0xffffffffu, t0 != m0 || t1 != m1)) {
            const float f0 = ex2(m0 - z0), f1 = ex2(m1 - z1);
            l0 *= f0; l1 *= f1;
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int u = 0; u < 2; ++u) { o[b][u][0] *= f0; o[b][u][1] *= f1; o[b][u][2] *= f0; o[b][u][3] *= f1; }
            m0 = t0; m1 = t1;
        }
        // weights, from (position g, columns 2 t, 2 t + 1) to (positions 2 t, 2 t + 1, column g)
        float p[2][4];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const float x = ex2(s[m][2 * u] - z0), y = ex2(s[m][2 * u + 1] - z1);
                l0 += x; l1 += y;
                const uint32_t xb = __float_as_uint(x), yb = __float_as_uint(y);
                const uint32_t hi = movmatrix(__byte_perm(xb, yb, 0x7632)), lo = movmatrix(__byte_perm(xb, yb, 0x5410));
                p[m][2 * u] = __uint_as_float(__byte_perm(lo, hi, 0x5410));
                p[m][2 * u + 1] = __uint_as_float(__byte_perm(lo, hi, 0x7632));
            }
        }
        // scales of the values, and the power of two that brings the largest product of the tile into [2^13, 2^14): of what column g sees,
        // as what lies behind must not change a bit
        const bool edge = j0 + TILE > base + col0 / a.group;
        const __half* vd = (const __half*)(at + 2 * S::KBYTES + S::DBYTES);
        float d[2][4][NB], top = 0.0f;
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                load_scales(vd + (16 * m + 2 * t + (u & 1) + 8 * (u >> 1)) * NB, d[m][u]);
                const bool out_of_sight = edge && j0 + 16 * m + 2 * t + (u & 1) + 8 * (u >> 1) >= seen_g;
#pragma unroll
                for (int b = 0; b < NB; ++b) top = fmaxf(top, out_of_sight ? 0.0f : fabsf(d[m][u][b]));
            }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int shift = plane_shift(top);
        const float up = exp2i(shift), down = exp2i(-shift);
        const float down0 = edge ? __shfl_sync(0xffffffffu, down, 8 * t) : down, down1 = edge ? __shfl_sync(0xffffffffu, down, 8 * t + 4) : down;
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int u = 0; u < 4; ++u) p[m][u] *= up;
        const uint32_t* vq = (const uint32_t*)(at + S::KBYTES);
        uint32_t w[4][NB];                        // pairs of positions t, t + 4, t + 8, t + 12
#pragma unroll
        for (int u = 0; u < 4; ++u) load_words(vq + (t + 4 * u) * (NB * 8) + g * NB, w[u]);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            float x[2][4] = {};
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                uint32_t h0, h1, r0, r1, e0[4], e1[4];
                planes_of(p[m][0] * d[m][0][b], p[m][1] * d[m][1][b], &h0, &r0);
                planes_of(p[m][2] * d[m][2][b], p[m][3] * d[m][3][b], &h1, &r1);
                levels_of(w[2 * m][b], e0);
                levels_of(w[2 * m + 1][b], e1);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const uint32_t f[4] = {e0[2 * u], e0[2 * u + 1], e1[2 * u], e1[2 * u + 1]};
                    mma16816(x[u], f, r0, r1);
                    mma16816(x[u], f, h0, h1);
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
    for (int w = 4; w < 32; w <<= 1) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, w);
        l1 += __shfl_xor_sync(0xffffffffu, l1, w);
    }
    if (g == 0) {
        warp_ml[warp][2 * t] = make_float2(m0, l0);
        warp_ml[warp][2 * t + 1] = make_float2(m1, l1);
    }
    float* const mo = (float*)ring;               // [column][channel]
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int ch = 32 * b + 16 * u + g;
            mo[2 * t * PAD + ch] = o[b][u][0];
            mo[(2 * t + 1) * PAD + ch] = o[b][u][1];
            mo[2 * t * PAD + ch + 8] = o[b][u][2];
            mo[(2 * t + 1) * PAD + ch + 8] = o[b][u][3];
        }
    __syncthreads();
    if (tid < SW * COLS) {
        const int col = tid % COLS;
        float m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int w = 0; w < SW; ++w) m = fmaxf(m, warp_ml[w][col].x);
        const float z = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int w = 0; w < SW; ++w) l += warp_ml[w][col].y * ex2(warp_ml[w][col].x - z);
        warp_f[tid / COLS][col] = ex2(warp_ml[tid / COLS][col].x - z);
        if (tid < COLS) cta_ml[col] = make_float2(m, l);
    }
    __syncthreads();
    float* const joined = (float*)fresh;          // the new rows in it have been read
    for (int e = tid; e < COLS * DIM; e += 32 * SW) {
        const int col = e / DIM, ch = e % DIM;
        float x = 0.0f;
#pragma unroll
        for (int w = 0; w < SW; ++w) x = fmaf(((const float*)(smem + w * (S::STAGES * S::BYTES)))[col * PAD + ch], warp_f[w][col], x);
        joined[col * PAD + ch] = x;
    }
    cg::cluster_group cluster = cg::this_cluster();
    if (cs > 1) cluster.sync();
    else __syncthreads();
    // every rank joins its share of the elements
    auto whole = [&](int col, float* z) {
        float m = -INFINITY, l = 0.0f;
        for (int r = 0; r < cs; ++r) m = fmaxf(m, cluster.map_shared_rank(cta_ml, r)[col].x);
        *z = m == -INFINITY ? 0.0f : m;
        for (int r = 0; r < cs; ++r) {
            const float2 x = cluster.map_shared_rank(cta_ml, r)[col];
            l = fmaf(x.y, ex2(x.x - *z), l);
        }
        return l;
    };
    for (int e = rank * (32 * SW) + tid; e < cols * DIM; e += cs * (32 * SW)) {
        const int col = e / DIM, ch = e % DIM;
        float z, x = 0.0f;
        const float l = whole(col, &z);
        for (int r = 0; r < cs; ++r) x = fmaf(cluster.map_shared_rank(joined, r)[col * PAD + ch], ex2(cluster.map_shared_rank(cta_ml, r)[col].x - z), x);
        out[place(col) + ch] = l == 0.0f ? 0.0f : x / l;
        if (ch == 0 && stats) stats[((size_t)first + (col0 + col) / a.group) * (c.n_kv * a.group) + h * a.group + (col0 + col) % a.group] = make_float2(z, l);
    }
    if (a.mass && !stats) {
        // the weights once more, against the whole row's maximum and sum: the last tile's scores are still there
        float z0, z1;
        l0 = whole(2 * t, &z0);
        l1 = whole(2 * t + 1, &z1);
        l0 = 2 * t < cols && l0 != 0.0f ? 1.0f / l0 : 0.0f;
        l1 = 2 * t + 1 < cols && l1 != 0.0f ? 1.0f / l1 : 0.0f;
        float* const mass = a.mass + ((size_t)seq * c.n_kv + h) * c.cap;
        if (cs > 1) cluster.sync();               // the ring may be written, and no rank leaves while it is read
        else __syncthreads();
        const int last = tiles > mine ? mine + (tiles - 1 - mine) / stride * stride : -1;
        for (int tile = last; tile >= 0; tile -= stride) {
            if (tile != last) {
                __syncwarp();
                ask<NB>(c, row0 + (size_t)tile * TILE, ring, lane, false);
                cp_commit();
                cp_wait<0>();
                __syncwarp();
                tile_scores<NB>(ring, qh, ql, inv0, inv1, tile * TILE, seen0, seen1, g, t, s);
            }
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    float x = (l0 != 0.0f ? ex2(s[m][2 * u] - z0) * l0 : 0.0f) + (l1 != 0.0f ? ex2(s[m][2 * u + 1] - z1) * l1 : 0.0f);
                    x += __shfl_xor_sync(0xffffffffu, x, 1);
                    x += __shfl_xor_sync(0xffffffffu, x, 2);
                    const int j = tile * TILE + 16 * m + 8 * u + g;
                    if (t == 0 && j < end) mass[j] = (j < (a.k ? len : end) ? mass[j] : 0.0f) + x;
                }
        }
        return;
    }
    if (cs > 1) cluster.sync();                   // no rank leaves while another reads its memory
}

template <int NB>
int launch_step_t(const Kv4& c, const Kv4Attend& a, const KvRows& rows, int groups, int cs, float2* stats, int device, cudaStream_t st) {
    using S = StepShape<NB>;
    static bool attr_set[64] = {};
    if (device >= 64 || !attr_set[device]) {
        FC_CUDA(cudaFuncSetAttribute(kv4_step_kernel<NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM));
        if (device < 64) attr_set[device] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(cs, c.n_kv * groups, c.n_seq);
    cfg.blockDim = dim3(32 * SW);
    cfg.dynamicSmemBytes = S::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cs;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    FC_CUDA(cudaLaunchKernelEx(&cfg, kv4_step_kernel<NB>, c, a, rows, stats));
    FC_LAUNCHED();
    return FC_OK;
}

}  // namespace

bool kv4_step_covers(const Kv4& c, int group, int max_rows) {
    return max_rows <= kStepRows && (long long)max_rows * group <= 64;
}

int launch_kv4_step(const Kv4& c, const Kv4Attend& a, const KvRows& rows, int max_rows, float2* stats, int device, cudaStream_t st) {
    const int groups = (max_rows * a.group + COLS - 1) / COLS;
    // as many CTAs as are resident, and no more than a tile for each warp of them
    const long long clusters = (long long)c.n_seq * c.n_kv * groups;
    const int most = (c.cap + TILE * SW - 1) / (TILE * SW);
    int cs = 1;
    while (cs < 8 && cs * 2 <= most && clusters * cs * 2 <= 296) cs *= 2;
    switch (c.nb) {
        case 1: return launch_step_t<1>(c, a, rows, groups, cs, stats, device, st);
        case 2: return launch_step_t<2>(c, a, rows, groups, cs, stats, device, st);
        case 3: return launch_step_t<3>(c, a, rows, groups, cs, stats, device, st);
        case 4: return launch_step_t<4>(c, a, rows, groups, cs, stats, device, st);
        case 5: return launch_step_t<5>(c, a, rows, groups, cs, stats, device, st);
        case 6: return launch_step_t<6>(c, a, rows, groups, cs, stats, device, st);
        case 7: return launch_step_t<7>(c, a, rows, groups, cs, stats, device, st);
        default: return launch_step_t<8>(c, a, rows, groups, cs, stats, device, st);
    }
}

}  // namespace fc
