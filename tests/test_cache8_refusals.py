"""Arguments of the calls over a cache in 8 bits that name no kernel are refused as such, on the host."""

import pytest

from atomserve_amd.kernels import ops
from tests.test_cache8 import nothing_is_launched, prompt, single  # noqa: F401 (a fixture that every test here uses)


@pytest.mark.parametrize("query_tiles", [0, 3, 4, -1])
def test_other_numbers_of_query_tiles_are_refused(query_tiles):
    with pytest.raises(ops.KernelError, match="query tiles"):
        prompt(query_tiles=query_tiles)


@pytest.mark.parametrize("query_tiles", [None, 1, 2])
def test_one_two_or_a_choice_go_to_the_kernel(query_tiles):
    with pytest.raises(AssertionError, match="would have been launched"):
        prompt(query_tiles=query_tiles)


@pytest.mark.parametrize("call", [single, prompt])
@pytest.mark.parametrize("out", [None, 3])
def test_results_that_are_no_tensor_are_refused(call, out):
    with pytest.raises(ops.KernelError):
        call(out=out)


def test_single_queries_without_heads_are_refused():
    with pytest.raises(ops.KernelError, match="heads 0/2"):
        single(H=0)


@pytest.mark.parametrize("wrong", [["--design", "dozusun"], ["--design", "tokuvik"], ["--dtype", "fp32"], ["--block-size", "8"]])
def test_a_benchmark_that_would_not_hold_its_cache_in_8_bits_is_refused(monkeypatch, capsys, wrong):
    import sys

    import bench

    monkeypatch.setattr(sys, "argv", ["bench.py", "--cache-bits", "8"])
    assert bench.parse_args().cache_bits == 8
    monkeypatch.setattr(sys, "argv", ["bench.py", *wrong])
    assert bench.parse_args().cache_bits == 0
    monkeypatch.setattr(sys, "argv", ["bench.py", "--cache-bits", "8", *wrong])
    with pytest.raises(SystemExit):
        bench.parse_args()
    assert "--cache-bits 8" in capsys.readouterr().err
