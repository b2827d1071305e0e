"""Scratch that is kept for a stream, and host threads that share the stream (no GPU: the library is played by a function)."""

import threading
import time

import pytest
import torch

from veloxquant_mlx_amd import _lib, kernels as K

CPU = torch.device("cpu")


@pytest.fixture
def scratch(monkeypatch):
    """Tables of this test alone, outside of any capture."""
    monkeypatch.setattr(K, "_capturing", lambda: False)
    monkeypatch.setattr(K, "_workspaces", {})
    monkeypatch.setattr(K, "_scratch_locks", {}, raising=False)


def _in_threads(*calls):
    failed = []

    def run(call):
        try:
            call()
        except BaseException as e:   # noqa: BLE001 (handed on to the test)
            failed.append(e)

    threads = [threading.Thread(target=run, args=(c,)) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not any(t.is_alive() for t in threads)
    if failed:
        raise failed[0]


def _library(mark, need, under_way):
    """A library call of two launches: the first writes into the scratch that it is handed, the second reads it."""
    def call(ws):
        if ws.numel() < need:
            return _lib.VQ_ERR_WORKSPACE
        under_way.append(mark)
        at_once.append(len(under_way))
        ws[:need] = mark
        time.sleep(0.002)   # (as the interpreter's lock is free while a library call runs)
        kept = any(t is ws for t in K._workspaces.values())
        right = kept and bool((ws[:need] == mark).all())
        under_way.remove(mark)
        assert right, "another call's launches came between, or its scratch took this one's place"
        return 0

    at_once: list[int] = []
    return call, at_once


def _calls(mark, need, stream, under_way, times=10):
    call, at_once = _library(mark, need, under_way)

    def go():
        for _ in range(times):
            assert K._scratch_call(CPU, stream, call, lambda ws: need, lambda ws, captured: ws) == 0

    return go, at_once


def test_calls_of_two_threads_on_one_stream_come_one_after_the_other(scratch):
    under_way = []
    a, at_once = _calls(1, 1000, 7, under_way)
    b, _ = _calls(2, (1 << 20) + 5, 7, under_way)       # (its first call takes larger scratch)
    _in_threads(a, b)
    assert max(at_once) == 1 and len(K._workspaces) == 1


def test_streams_do_not_wait_for_each_other(scratch):
    both = threading.Barrier(2, timeout=30)

    def call(ws):
        both.wait()      # (each waits until the other one's call runs too)
        return 0

    _in_threads(*(lambda stream=stream: K._scratch_call(CPU, stream, call, lambda ws: 0, lambda ws, captured: ws) for stream in (7, 8)))


def test_every_fetch_of_kept_scratch_is_under_the_lock():
    """Each function that fetches the scratch kept for a stream does so inside the stream's lock, launch included."""
    import ast
    import inspect
    tree = ast.parse(inspect.getsource(K))
    fetched = 0
    for f in tree.body:
        if not isinstance(f, ast.FunctionDef) or f.name in ("_workspace", "_scratch_lock"):
            continue
        locked = set()
        for w in ast.walk(f):
            if isinstance(w, ast.With) and any(isinstance(i.context_expr, ast.Call) and getattr(i.context_expr.func, "id", "") == "_scratch_lock" for i in w.items):
                locked |= {id(x) for x in ast.walk(w)}
        for c in ast.walk(f):
            if isinstance(c, ast.Call) and getattr(c.func, "id", "") == "_workspace":
                fetched += 1
                assert id(c) in locked, f"{f.name}, line {c.lineno}"
    assert fetched >= 6
