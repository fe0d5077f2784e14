"""A refused call leaves nothing behind: the HIP runtime keeps a thread's last error until it is asked for it, and
a launch's check (this library's, or torch's) takes what it finds there for the launch's own."""
import ctypes as C

import numpy as np
import pytest
import torch

from dizo_amd import _lib as L
from dizo_amd import token_loss as T
from dizo_amd._lib import DzError
from dizo_amd.table import ZOTable, stream_handle

pytestmark = pytest.mark.gpu

HOST = np.zeros(4096, dtype=np.float32)  # memory that the device's allocator does not know


def _score(at):
    out, t = torch.zeros(8, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    L.call("dz_token_logprobs", at, L.DZ_DTYPE_F32, 1, 4, 16, 0, 16, t.data_ptr(), 0, 1, -100, 0, out.data_ptr(), out[4:].data_ptr(), None, None,
           None, 0, 0, None, 0, 0, None, 0, 0, stream_handle())


def _distill(at):
    out, t = torch.zeros(4, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    L.call("dz_topk_distill", at, L.DZ_DTYPE_F32, 1, 4, 16, 0, 16, out.data_ptr(), t.data_ptr(), 1, 1.0, 1, out.data_ptr(), None, 0, 0, None, 0, 0,
           stream_handle())


def _head(at):
    out, t = torch.zeros(8, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    work = torch.zeros(1 << 16, dtype=torch.uint8, device="cuda")
    L.call("dz_linear_token_logprobs", at, at, L.DZ_DTYPE_F32, 4, 16, 16, 16, 16, t.data_ptr(), -100, out.data_ptr(), out[4:].data_ptr(),
           work.data_ptr(), work.numel(), stream_handle())


def _table(at):
    table = C.c_void_p()
    L.call("dz_table_create", (C.c_uint64 * 1)(at), None, (C.c_int64 * 1)(8), None, 1, L.DZ_DTYPE_F32, 0, C.byref(table))


def _norms(at):
    out = torch.zeros(1, dtype=torch.float64, device="cuda")
    L.call("dz_group_sumsq_static", (C.c_uint64 * 1)(at), (C.c_uint64 * 1)(at), (C.c_int64 * 1)(8), 1, L.DZ_DTYPE_F32, out.data_ptr(), None, None,
           stream_handle())


@pytest.mark.parametrize("refused", [_score, _distill, _head, _table, _norms], ids=["token_logprobs", "topk_distill", "head", "table", "norms"])
def test_the_call_after_a_refused_one_works(refused):
    x, t = torch.randn(4, 16, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    want = T.token_logprobs(x, t).logprobs
    for after in (lambda: T.token_logprobs(x, t).logprobs, lambda: want + 0, lambda: ZOTable([x]).close()):
        with pytest.raises(DzError, match="not device memory"):
            refused(HOST.ctypes.data)
        got = after()
        assert got is None or torch.equal(got, want)
