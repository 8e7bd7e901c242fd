"""The model-level benchmark with rotary positions: both backends agree."""

import pytest
import torch

from flashbob_b200 import hvp_bench


def _rows(argv):
    return hvp_bench.run(hvp_bench.build_parser().parse_args(argv))


def test_both_backends_agree_on_the_cpu():
    rows = _rows("--seq-lens 16 33 --dim 32 --heads 2 --layers 2 --warmup 0 --iters 1 --dtype fp32 --device cpu --rotary".split())
    plain = _rows("--seq-lens 16 --dim 32 --heads 2 --layers 2 --warmup 0 --iters 1 --dtype fp32 --device cpu".split())
    # fp32 throughout, sums in another order
    assert all(r["hv_l2_rel"] < 1e-4 for r in rows + plain)


@pytest.mark.gpu
@pytest.mark.parametrize("argv", ["--dim 128 --heads 2", "--dim 256 --heads 4 --kv-heads 2"])
def test_both_backends_agree_on_the_gpu(argv):
    rows = _rows(f"--seq-lens 128 300 --layers 1 --warmup 1 --iters 2 --rotary {argv}".split())
    # bf16: both round every operand, probability and gradient of the chain, a dozen roundings of 2^-9 on average in
    # quadrature on either side, and the materialized one its scores too
    assert all(r["hv_l2_rel"] < 0.03 for r in rows)
