"""Symmetric operands of the row collectives in tests: a matrix per PE, possibly with padded rows and
an odd start, every byte of which is known before a call and looked at after it."""
import numpy as np

import roc_shmem_amd as rs

FILL = 0x5A


class Rows:
    """rows x cols elements on every PE, `ld` elements from row to row, `shift` elements into an
    allocation that is otherwise full of FILL bytes."""

    def __init__(self, rows, cols, np_dtype, ld=None, shift=0, slack=8):
        self.rows, self.cols, self.ld, self.shift = rows, cols, ld or cols, shift
        self.dtype = np.dtype(np_dtype)
        n = shift + max(rows - 1, 0) * self.ld + (cols if rows else 0) + slack
        self.whole = rs.sym_array(n, self.dtype, fill=FILL)
        self.addr = self.whole.addr + shift * self.dtype.itemsize
        self.before = {}

    def _matrix(self, flat):
        return np.lib.stride_tricks.as_strided(flat[self.shift:], (self.rows, self.cols),
                                               (self.ld * self.dtype.itemsize, self.dtype.itemsize))

    def write(self, pe, values):
        flat = self.whole.read(pe)
        self._matrix(flat)[:] = values
        self.whole.write(pe, flat)
        return self

    def write_all(self, per_pe):
        for pe, v in enumerate(per_pe):
            self.write(pe, v)
        return self

    def remember(self):
        self.before = {pe: self.whole.read(pe).copy() for pe in range(rs.roc_shmem_n_pes())}

    def read(self, pe):
        return self._matrix(self.whole.read(pe)).copy()

    def check_rest(self, pe, name, written_rows):
        """Outside the first `written_rows` rows every byte is what it was before."""
        now, was = self.whole.read(pe), self.before[pe].copy()
        self._matrix(was)[:written_rows] = self._matrix(now)[:written_rows]
        assert np.array_equal(now.view(np.uint8), was.view(np.uint8)), "%s: PE %d: bytes beyond the result changed" % (name, pe)
