"""DecodeEngine called from other streams than its own: order, lifetime of the caller's tensors, capture."""

import numpy as np
import pytest
import torch

from gemmagemini4hackathon2026_10_2425_b200.engine import DecodeEngine, make_block_table
from gemmagemini4hackathon2026_10_2425_b200.tp import ModelShape

pytestmark = pytest.mark.gpu
DEV = "cuda"
B, MAX_CTX, BLOCKS = 3, 256, 64
SLEEP = 20_000_000  # cycles: about 10 ms


class Case:
    """A small engine, inputs of a step on the CPU, and the step's logits from the engine's own stream."""

    def __init__(self):
        self.eng = DecodeEngine(ModelShape(256, 2, 4, 2, 64, 512, 1000, 1e-5, 10000.0), max_batch=B, max_ctx=MAX_CTX, n_blocks=BLOCKS)
        self.eng.alloc_kv(fill_seed=1)
        self.eng.random_weights(2, std=0.05)
        r = np.random.default_rng(3)
        self.lens = [40, 100, 7]
        table = make_block_table(self.lens, MAX_CTX // 16, BLOCKS, seed=4)
        self.host = [torch.from_numpy(r.integers(0, 1000, B).astype(np.int32)), torch.tensor(self.lens, dtype=torch.int32), table.int()]
        torch.cuda.synchronize()
        with torch.cuda.stream(self.eng.stream):
            ins = [t.to(DEV) for t in self.host]
            nxt, self.want = self.outputs()
            self.eng.step(*ins, nxt, self.want, use_graph=False)
        torch.cuda.synchronize()
        self.next = nxt

    def outputs(self):
        return torch.zeros(B, dtype=torch.int32, device=DEV), torch.zeros(B, self.eng.lm_rows, device=DEV)

    def check(self, nxt, logits):
        assert torch.equal(logits, self.want) and torch.equal(nxt, self.next)


@pytest.fixture(scope="module")
def case():
    c = Case()
    yield c
    c.eng.close()


@pytest.mark.parametrize("use_graph", [False, True])
def test_step_waits_for_the_callers_stream(case, use_graph):
    """Inputs that are still being made on the caller's stream when the step is called."""
    ins = [torch.zeros_like(t, device=DEV) for t in case.host]
    pinned = [t.pin_memory() for t in case.host]
    nxt, logits = case.outputs()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(SLEEP)
        for d, h in zip(ins, pinned):
            d.copy_(h, non_blocking=True)
        case.eng.step(*ins, nxt, logits, use_graph=use_graph)
    case.eng.stream.synchronize()
    case.check(nxt, logits)


def test_tensors_of_a_queued_step_are_not_handed_out_again(case):
    """The caller drops its inputs while the engine's stream is still busy and makes others of that size."""
    nxt, logits = case.outputs()
    torch.cuda.synchronize()
    with torch.cuda.stream(case.eng.stream):
        torch.cuda._sleep(SLEEP)
    ins = [t.to(DEV) for t in case.host]
    case.eng.step(*ins, nxt, logits, use_graph=False)
    del ins
    junk = [torch.full_like(t, 1, device=DEV) for t in case.host for _ in range(4)]
    case.eng.stream.synchronize()
    case.check(nxt, logits)
    del junk


@pytest.mark.parametrize("own", [False, True])
@pytest.mark.parametrize("use_graph", [False, True])
def test_step_in_a_callers_capture(case, own, use_graph):
    """A step captured on another stream (or the engine's own, without a graph of its own) is part of the
    caller's graph: work captured behind it follows it, replays read the inputs anew, and the engine goes on."""
    if own and use_graph:
        pytest.skip("a graph of its own is captured on the engine's stream")
    ins = [t.to(DEV) for t in case.host]
    nxt, logits = case.outputs()
    copy = torch.zeros_like(logits)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=case.eng.stream if own else torch.cuda.Stream()):
        case.eng.step(*ins, nxt, logits, use_graph=use_graph)
        copy.copy_(logits)
    assert logits.eq(0).all()  # captured, not run
    for _ in range(2):
        logits.zero_(), nxt.zero_(), copy.zero_()
        g.replay()
        torch.cuda.synchronize()
        case.check(nxt, logits)
        assert torch.equal(copy, logits)
    ins[0].zero_()
    g.replay()
    torch.cuda.synchronize()
    assert not torch.equal(logits, case.want)
    logits.zero_()
    case.eng.step(*[t.to(DEV) for t in case.host], nxt, logits)
    case.eng.stream.synchronize()
    case.check(nxt, logits)
    del g


def test_generate_in_a_callers_capture_is_refused(case):
    ins = [t.to(DEV) for t in case.host]
    ring, count = torch.zeros(4, B, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    x = torch.zeros(4, device=DEV)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        x += 1
        with pytest.raises(ValueError, match="capture step"):
            case.eng.generate(*ins, 2, ring, count)
        x += 1
    g.replay()
    torch.cuda.synchronize()
    assert x.eq(2).all() and ring.eq(0).all()
    del g
    case.eng.generate(*ins, 2, ring, count)
    case.eng.stream.synchronize()
    assert count.item() == 2 and torch.equal(ring[0], case.next)
