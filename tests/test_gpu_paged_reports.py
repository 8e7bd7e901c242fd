"""An error that the GPU found is raised once: calls after it are not told of it again, whatever of the faulty call still runs."""

import pytest
import torch

import paged_reference as R
from flashbob_b200 import _lib, ops
from flashbob_b200.paged import append_kv, read_kv, sdpa_paged
from test_gpu_paged import _cache, _heads

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("what", ["attention", "tiles", "append", "read"])
@pytest.mark.parametrize("fault", ["page", "length"])
def test_one_faulty_call_is_one_error(bits, what, fault):
    """The faulty call's own look at the status may fall between two of its reports, of several kernels or threads."""
    n = 4000
    seqs = R.Sequences([n, n, n], 16)
    cache = _cache(seqs, 4, 64, torch.bfloat16, bits, garbage=False)
    N = {"attention": 2, "tiles": 700, "append": 3000, "read": 0}[what]
    x = None if what == "read" else _heads((3, 4, N, 64), torch.bfloat16, 1)
    call = {"attention": lambda: sdpa_paged(x, cache, seqs.table, seqs.lengths), "tiles": lambda: sdpa_paged(x, cache, seqs.table, seqs.lengths),
            "append": lambda: append_kv(x, x, cache, seqs.table, seqs.lengths), "read": lambda: read_kv(cache, seqs.table, seqs.lengths, n)}[what]
    good = (seqs.table.clone(), seqs.lengths.clone())
    wrong = (good[0].clone(), good[1].clone())
    if fault == "page":
        wrong[0][1, 200:] = 1 << 30
    else:
        wrong[1][:2] = 1 << 30
    before, ops._CHECK_STATUS = ops._CHECK_STATUS, False
    try:
        call()
        torch.cuda.synchronize()
        for _ in range(60):
            seqs.table.copy_(wrong[0])
            seqs.lengths.copy_(wrong[1])
            raised = 0
            try:
                call()
            except _lib.BobSm100Error:
                raised = 1
            torch.cuda.synchronize()
            seqs.table.copy_(good[0])
            seqs.lengths.copy_(good[1])
            if not raised:
                with pytest.raises(_lib.BobSm100Error):
                    call()
            call()
            torch.cuda.synchronize()
            call()
    finally:
        ops._CHECK_STATUS = before
