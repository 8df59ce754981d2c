// The key / value cache of 4-bit levels: its layout in device memory, shared by the kernels that fill, read, attend to and
// compact it.
//
// A row of head_dim values (one position, one key / value head) is cut into blocks of 32 (`nb` of them). A block is an f16
// scale d = f16(m / -8), m its value of largest magnitude, and levels clamp(rint(x / d), -8, 7), stored plus 8 as nibbles: 4.5
// bits a value. Rows of a (sequence, head) lie one after the other, so that a head's positions are read as one stream.
// The order inside a row is that of the matrix fragments which read it (a lane is (g, t) = (lane / 4, lane % 4)):
//   keys    word t * nb + b of a row: nibble i holds channel 32 b + 8 t + i. The contraction runs over channels, nibbles 4 bits
//           apart (i, i + 4) are a fragment's pair of neighbours, and a lane's words of all blocks are contiguous.
//   values  word g * nb + b of a PAIR of rows: nibble j of the low half holds channel 32 b + 8 j + g of the even row, nibble j of
//           the high half that of the odd row. The contraction runs over positions, so the pair of neighbours is two rows.
//   scales  [row][nb] f16, keys and values apart.
// Rows are padded to a multiple of 64 a (sequence, head), zeroed at creation: a tile may be read past the last position.
#pragma once
#include "fc_common.cuh"

namespace fc {

constexpr int kKvBlock = 32;
constexpr int kKvTile = 64;        // rows a (sequence, head) is padded to a multiple of
constexpr int kKvMaxSeq = 256;

struct Kv4 {
    uint32_t *kq, *vq;
    __half *kd, *vd;
    int n_seq, n_kv, nb, cap, cap_pad;
    __host__ __device__ size_t row(int seq, int head, int pos) const { return ((size_t)seq * n_kv + head) * cap_pad + pos; }
    __host__ __device__ int dim() const { return nb * kKvBlock; }
};

// Where each sequence's new rows begin among the packed rows of a call; n_seq + 1 entries.
struct KvRows { int start[kKvMaxSeq + 1]; };

}  // namespace fc

struct fc_kv4 {
    int device = 0;
    fc::Kv4 c{};
    fc::Arena arena;
};
