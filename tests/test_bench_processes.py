"""bench.py's CPU baseline: how many worker processes it starts.  Each opens the GPU (torch's autograd engine asks for the device count), which 16 processes at most
may hold at once, bench.py's own among them."""
import os
import types

import numpy as np

import bench


def test_the_cpu_baseline_starts_few_processes_on_a_host_of_many_cores(monkeypatch):
    started = []

    class Pool:
        def __init__(self, procs):
            started.append(procs)

        def __enter__(self):
            return self

        def __exit__(self, *exc):
            pass

        def map(self, f, jobs):
            return [f(j) for j in jobs]

    import multiprocessing
    monkeypatch.setattr(multiprocessing, "get_context", lambda method: types.SimpleNamespace(Pool=Pool))
    monkeypatch.setattr(os, "cpu_count", lambda: 256)
    monkeypatch.setattr(bench, "_oracle_worker", lambda args: [(k, 0.5, np.zeros((3, 3)), np.zeros(4)) for k, _ in args[0]])
    sample = [(k, types.SimpleNamespace(adj=np.zeros((3, 3)))) for k in range(32)]
    base, _, res = bench.cpu_baselines(types.SimpleNamespace(ck={"sd": {}}, targets=range(400)), sample, 1)
    assert started == [base["cores"]] and 1 + started[0] < 16
    assert sorted(res) == list(range(32))                      # every target of the sample, by whichever worker
    assert bench.oracle_processes(3) == 3 and bench.oracle_processes(1000) == started[0]
    monkeypatch.setattr(os, "cpu_count", lambda: 2)
    assert bench.oracle_processes(32) == 2


def test_no_other_pool_is_sized_by_the_hosts_cores():
    source = open(bench.__file__).read()
    assert source.count(".Pool(") == source.count("procs = oracle_processes(") == 2
