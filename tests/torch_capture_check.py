"""Run by tests/test_gpu_borrowed.py in a process of its own: a step of a search recorded into one of torch's graphs, replayed over new inputs with eager work, of
torch and of this library, and waits between the replays; and two graphs, each with a selection of its own, replayed one after the other."""
import os
import sys

import numpy as np
import torch

torch.cuda.init()
sys.path[:0] = [os.path.dirname(os.path.dirname(os.path.abspath(__file__))), os.path.dirname(os.path.abspath(__file__))]
import arrow_gpu_amd as ag  # noqa: E402
import rows_ref as R  # noqa: E402

dev = ag.GpuDevice(torch.cuda.current_device())
side = torch.cuda.Stream()
rng = np.random.default_rng(0)
f32 = lambda a: torch.from_numpy(np.asarray(a, np.float32)).cuda()  # noqa: E731
i32 = lambda a: torch.from_numpy(np.asarray(a, np.int32)).cuda()  # noqa: E731
rows = lambda t: ag.RowsGPU.of_tensor(t, dev)  # noqa: E731
u32 = lambda t: ag.UInt32ArrayGPU.of_tensor(t, dev)  # noqa: E731
N, HEADS, DIM, GROUP, BEAMS, VOCAB = 8, 2, 64, 32, 4, 1003


class Step:
    def __init__(self):
        self.x, self.logits, self.scores, self.state = f32(np.zeros((N, HEADS, DIM))), f32(np.zeros((N, VOCAB))), f32(np.zeros(N)), f32(np.zeros((N, 3, 5, 8)))
        self.slots = i32(rng.permutation(20)[:N])
        self.codes, self.scales = torch.zeros((20, HEADS, DIM), dtype=torch.uint8, device="cuda"), f32(np.zeros((20, HEADS, DIM // GROUP)))
        self.back, self.moved = torch.zeros_like(self.x), torch.zeros_like(self.state)
        self.found = [torch.zeros((N // BEAMS, BEAMS), dtype=t, device="cuda") for t in (torch.float32, torch.int32, torch.int32)]
        self.store = ag.QuantisedRowsGPU.of_tensors(self.codes, self.scales, dev, code="i8", heads=HEADS, dim=DIM, group=GROUP)
        self.selection = ag.BeamSelection.of_tensors(*self.found, dev)

    def run(self, pipe):
        ag.put_quantised_op(self.store, rows(self.x), u32(self.slots), pipe)
        ag.take_quantised_op(self.store, u32(self.slots), pipe, out=rows(self.back))
        ag.select_beams_op(rows(self.logits), BEAMS, BEAMS, pipe, scores=ag.Float32ArrayGPU.of_tensor(self.scores, dev), out=self.selection)
        ag.take_rows_op(rows(self.state), self.selection.parents, pipe, out=rows(self.moved))

    def fill(self):
        self.given = [rng.standard_normal(t.shape).astype(np.float32) for t in (self.x, self.logits, self.scores, self.state)]
        for t, v in zip((self.x, self.logits, self.scores, self.state), self.given):
            t.copy_(torch.from_numpy(v))
        for t in (self.back, self.moved, *self.found):
            t.zero_()

    def check(self):
        x, logits, scores, state = self.given
        want = R.values(*R.quantise(x, "i8", GROUP), "i8", GROUP)
        assert (np.abs(self.back.cpu().numpy() - want) <= np.abs(want) * R.HALF_STEP["f32"] * 1.001).all()
        picks = R.select(logits.astype(np.float64), BEAMS, BEAMS, scores)
        assert np.array_equal(self.found[1].cpu().numpy(), picks[1]) and np.array_equal(self.found[2].cpu().numpy(), picks[2])
        assert np.array_equal(self.moved.cpu().numpy(), state[picks[1].reshape(-1)])


pipe = ag.ArrowComputePipeline(dev, "captured", hip_stream=side.cuda_stream)
steps, graphs = [Step(), Step()], []
with torch.cuda.stream(side):
    for s in steps:
        s.fill()
        s.run(pipe)  # once before the capture: the selection's workspace is there
        side.synchronize()
        s.check()
for s in steps:
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        s.run(pipe)
        try:
            ag.take_rows(rows(s.state), s.selection.parents, out=rows(s.moved))
        except ag.ArrowErrorGPU as e:
            assert "captures" in str(e)
        else:
            raise AssertionError("a call that waits was taken during a capture")
    graphs.append(g)
print("captured", flush=True)
for turn in range(5):
    for s, g in zip(steps, graphs):
        s.fill()
        g.replay()
        s.check()
    eager = ag.select_beams(rows(steps[0].logits), BEAMS, BEAMS, scores=ag.Float32ArrayGPU.of_tensor(steps[0].scores, dev))  # on torch's current stream
    assert np.array_equal(eager.values()[1], steps[0].found[1].cpu().numpy())
    assert float(torch.ones(100000, device="cuda").sum()) == 100000.0
    for s in steps:  # both in flight, nothing between them
        s.fill()
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    for s in steps:
        s.check()
pipe.sync()
print("torch capture OK")
