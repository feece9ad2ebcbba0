"""Selections of several host threads on one stream."""
import threading
import time
from types import SimpleNamespace

import pytest
import torch

import beam_plain as plain
from inferloop_b200.csrc import ops


def in_threads(calls):
    """Run the functions, a thread each, and raise what any of them raised."""
    wrong, start = [], threading.Barrier(len(calls))

    def run(call):
        try:
            start.wait()
            call()
        except BaseException as e:
            wrong.append(e)
    threads = [threading.Thread(target=run, args=(c,)) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    if wrong:
        raise wrong[0]


def test_calls_that_run_at_once_have_different_scratch(monkeypatch):
    """Without a device: while one call's launches are on their way to the stream, no other call is given its scratch."""
    using, taken = {}, []

    def launches(index, module, fn, *args):
        scratch = args[12]
        assert scratch not in using, "two selections write one scratch"
        using[scratch] = True
        taken.append(scratch)
        time.sleep(0.002)
        del using[scratch]
    monkeypatch.setattr(ops, "_ready", lambda *a: True)
    monkeypatch.setattr(ops, "_recording", lambda: False)
    monkeypatch.setattr(ops, "_call_on", launches)
    monkeypatch.setattr(ops, "_BEAM_SCRATCH", {})
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 7, raising=False)

    def call(vocab):
        x = torch.zeros(4, vocab)
        logits = SimpleNamespace(get_device=lambda: 0, dim=x.dim, shape=x.shape, stride=x.stride, data_ptr=x.data_ptr, dtype=x.dtype, device=x.device)
        i, f = torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, 4)
        ops.beam_select(logits, f, i, i, f)
    in_threads([lambda: [call(100) for _ in range(20)], lambda: [call(9000 + 4000 * n) for n in range(20)]])
    assert len(taken) == 40


@pytest.mark.gpu
def test_two_threads_on_one_stream():
    R, W, k, dev = 3, 4, 8, "cuda:0"
    cases = []
    for seed, vocab in ((1, 50000), (2, 50000), (3, 31000)):
        x = 3 * torch.randn(R * W, vocab, generator=torch.Generator().manual_seed(seed))
        scores = -5 * torch.rand(R, W, generator=torch.Generator().manual_seed(seed))
        cases.append((x.to(dev), scores.to(dev), plain.select(x, scores, k)[0]))
    outs = [[[torch.zeros(R, k, dtype=torch.int32, device=dev), torch.zeros(R, k, dtype=torch.int32, device=dev), torch.zeros(R, k, device=dev)]
             for _ in range(200)] for _ in cases]
    torch.cuda.synchronize()

    def calls(case, out):
        def run():
            for o in out:
                ops.beam_select(case[0], case[1], *o)
        return run
    in_threads([calls(c, o) for c, o in zip(cases, outs)])
    torch.cuda.synchronize()
    for (_, _, found), out in zip(cases, outs):
        for parents, tokens, _ in out:
            assert parents.tolist() == [f[0] for f in found] and tokens.tolist() == [f[1] for f in found]
