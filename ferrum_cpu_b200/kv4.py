"""The key / value cache of 4-bit levels (fc_kv4_*): filled, attended to, read back and cut down to a budget by the attention
weight that its positions have received. Arguments named *_ptr are device addresses; every call returns before its kernels run.
"""
import ctypes as C

from . import _lib
from ._lib import check


def row_counts(rows):
    """How many rows each sequence brings to a call, as the calls take it: made once where the numbers stay."""
    return (C.c_int32 * len(rows))(*rows)


class Kv4Cache:
    """n_seq sequences of up to `capacity` positions on one GPU. The lengths belong to the caller (device int32 [n_seq])."""

    def __init__(self, n_seq, n_kv_head, head_dim, capacity, device=0):
        self._h = C.c_void_p()
        self.n_seq, self.n_kv_head, self.head_dim, self.capacity, self.device = n_seq, n_kv_head, head_dim, capacity, device
        L = _lib.lib()
        check(L.fc_kv4_create(device, n_seq, n_kv_head, head_dim, capacity, C.byref(self._h)))
        self._attend, self._read, self._evict = L.fc_kv4_attend_dev, L.fc_kv4_read_dev, L.fc_kv4_evict_dev   # a short step takes less time than two lookups

    def _rows(self, rows):
        if rows is None or isinstance(rows, C.Array):
            counts = rows
        else:
            counts = row_counts(rows)
        if counts is not None and len(counts) != self.n_seq:
            raise _lib.FerrumCudaError(_lib.FC_E_SHAPE, f"rows of {len(counts)} sequences, the cache has {self.n_seq}")
        return counts

    def append_dev(self, k_ptr, v_ptr, ldkv, lens_ptr, rows=None, stream=None):
        check(_lib.lib().fc_kv4_append_dev(self._h, k_ptr, v_ptr, ldkv, self._rows(rows), lens_ptr, stream))

    def attend_dev(self, q_ptr, ldq, n_head, lens_ptr, out_ptr, ldo, k_ptr=None, v_ptr=None, ldkv=0, rows=None, scale=0.0, mass_ptr=None,
                   stream=None):
        """Causal attention of the rows' query heads; with k_ptr and v_ptr the rows go into the cache first."""
        rc = self._attend(self._h, q_ptr, ldq, n_head, k_ptr, v_ptr, ldkv, self._rows(rows), lens_ptr, scale, mass_ptr, out_ptr, ldo, stream)
        if rc:
            check(rc)

    def read_dev(self, n, k_ptr, v_ptr, from_ptr=None, stream=None):
        """What n positions of every sequence stand for, from from_ptr[s] on: f32 [n_seq][n][n_kv_head][head_dim]."""
        rc = self._read(self._h, from_ptr, n, k_ptr, v_ptr, stream)
        if rc:
            check(rc)

    def evict_dev(self, dst, lens_ptr, lens_out_ptr, budget, recent, mass_ptr, mass_out_ptr=None, kept_ptr=None, stream=None):
        """The last `recent` positions and the heaviest others, `budget` in all, to the cache `dst`."""
        rc = self._evict(self._h, dst._h, lens_ptr, lens_out_ptr, budget, recent, mass_ptr, mass_out_ptr, kept_ptr, stream)
        if rc:
            check(rc)

    def close(self):
        if self._h:
            _lib.lib().fc_kv4_free(self._h)
            self._h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
