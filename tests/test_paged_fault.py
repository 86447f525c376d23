"""The flag that a wrong index raises: read and cleared in one step, whatever other streams and threads do meanwhile."""

import threading

import pytest
import torch

import libcertex_b200 as certex
from libcertex_b200 import paged

gpu = pytest.mark.gpu


def test_the_library_refuses_what_has_no_flag_or_answer(built_library):
    cache = dict(keys=64, values=64, k0=64, k1=64, k2=64, v0=64, v1=64, v2=64, n_pages=1, page_size=1, kv=1, dim=8, dtype=0, fault=64)
    take = built_library.certexB200PagedTakeFault
    for args, text in (((None, 64), b"null cache"), ((paged._CACHE.pack(*{**cache, "fault": 0}.values()), 64), b"null cache"),
                       ((paged._CACHE.pack(*cache.values()), None), b"null answer"), ((paged._CACHE.pack(*cache.values()), 64), b"null resources")):
        assert take(None, *args) == 0 and text in built_library.cuvsGetLastErrorText()


def small():
    cache = certex.PagedCache(2, 4, 1, 8, dtype=torch.float32)
    q, table = torch.zeros((1, 1, 8), device="cuda"), torch.zeros((1, 1), device="cuda", dtype=torch.int32)
    wrong, right = (torch.tensor([n], device="cuda", dtype=torch.int32) for n in (5, 4))  # the table holds four tokens
    return cache, (lambda: cache.attend(q, table, wrong)), (lambda: cache.attend(q, table, right))


@gpu
def test_a_wrong_index_is_told_once():
    cache, wrong, right = small()
    right()
    assert not cache.faulted()
    wrong()
    right()
    assert cache.faulted() and not cache.faulted()


@gpu
def test_what_comes_while_the_flag_is_read_is_told_the_next_time(monkeypatch):
    """A call of another stream finds a wrong index right after the flag was read on the host."""
    cache, wrong, _ = small()
    wrong()
    side, read = torch.cuda.Stream(), torch.Tensor.item

    def item(t):
        v = read(t)
        monkeypatch.setattr(torch.Tensor, "item", read)
        with torch.cuda.stream(side):
            wrong()
        side.synchronize()
        return v

    monkeypatch.setattr(torch.Tensor, "item", item)
    assert cache.faulted()
    assert cache.faulted() and not cache.faulted()


@gpu
def test_no_report_is_lost_among_threads():
    """Threads with streams of their own: each waits for its wrong call and asks, so somebody is told of every round."""
    cache, wrong, _ = small()
    rounds, told = 50, [0] * 4
    gate = threading.Barrier(4)

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(rounds):
                gate.wait(60)
                wrong()
                torch.cuda.current_stream().synchronize()
                told[i] += cache.faulted()
                gate.wait(60)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    torch.cuda.synchronize()
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert sum(told) >= rounds and not cache.faulted()
