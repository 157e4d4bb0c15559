"""What is known about patterns, read by operators and written by Python from several threads at once."""
import threading

import pytest
import torch

from _util import to_dev
from intrasm_engine_amd import workloads as W
from intrasm_engine_amd.pytorch import ops as pyops

pytestmark = pytest.mark.gpu
ops = torch.ops.iex_ops


def test_tables_taken_while_notes_are_written(dev):
    """Operators take a pattern's tables, which only its Python object holds, while other threads write notes with the interpreter's lock in hand:
    nobody waits for somebody who waits for them."""
    pattern, q, k, _ = W.config3(heads=8)
    ri, _, ro, ci = to_dev(pattern, dev)
    q, k = (torch.from_numpy(x).to(dev).half() for x in (q, k))
    want = ops.sddmm_sputnik_half(q, k, ri, ro, ci)
    assert torch.equal(ops.sddmm_sputnik_half(q, k, ri, ro, ci), want) and ci.__dict__["_iex_csr"][7] is not None
    torch.cuda.synchronize()
    wrong, done = [], threading.Event()

    def read():
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(200):
                got = ops.sddmm_sputnik_half(q, k, ri, ro, ci)
            stream.synchronize()
            if not torch.equal(got, want):
                wrong.append(got)

    def write():
        offsets, columns = ro.clone(), ci.clone()
        while not done.is_set():
            pyops.mark_canonical(offsets, columns, pattern.k, measure=False)

    readers, writers = [threading.Thread(target=read, daemon=True) for _ in range(3)], [threading.Thread(target=write, daemon=True) for _ in range(2)]
    for t in readers + writers:
        t.start()
    for t in readers:
        t.join(60)
    stuck = any(t.is_alive() for t in readers)
    done.set()
    for t in writers:
        t.join(10)
    assert not stuck and not wrong
