"""The suite's protocol: a row's buffer sets are past twice the last-level cache, so that
no pass finds its inputs there. The library and the clock are stand-ins on the CPU."""

import pytest
import torch

from flint_amd import bench_suite


class Library:
    """Calls that note which bytes they were given."""

    def __init__(self):
        self.seen = {}

    def __getattr__(self, name):
        def call(*args, **kwargs):
            for t in (*args, *kwargs.values()):
                if isinstance(t, torch.Tensor):
                    self.seen[t.data_ptr()] = t.numel() * t.element_size()
            return 64      # what a size query returns

        return call


@pytest.mark.parametrize("row", ["flint_rotary", "flint_gemm_nt_gated", "flint_gemm_nn_dgated"])
def test_a_pass_over_the_sets_exceeds_twice_the_cache(monkeypatch, tmp_path, row):
    cache = 8 << 20
    monkeypatch.setattr(bench_suite, "M", 256)
    monkeypatch.setattr(bench_suite, "CACHE", cache)
    library, passes = Library(), []

    def clock(torch_, fn, sets, **_):
        library.seen.clear()
        for st in sets:
            fn(st)
        passes.append(sum(library.seen.values()))
        return 1.0

    monkeypatch.setattr(bench_suite, "_time_gpu", clock)
    rows = bench_suite.run(library, torch, torch.device("cpu"), tmp_path / "suite.json", only=row)
    assert len(passes) == len(rows) >= 1
    assert all(seen >= 2 * cache for seen in passes), passes
