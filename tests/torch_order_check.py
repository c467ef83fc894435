"""Run by tests/test_gpu_borrowed.py in a process of its own: calls that take no pipeline, over tensors that torch is still computing when they are made, and
that torch overwrites right behind them."""
import os
import sys

import numpy as np
import torch

torch.cuda.init()
sys.path[:0] = [os.path.dirname(os.path.dirname(os.path.abspath(__file__))), os.path.dirname(os.path.abspath(__file__))]
import arrow_gpu_amd as ag  # noqa: E402
import rows_ref as R  # noqa: E402

dev = ag.GpuDevice(torch.cuda.current_device())
busy = torch.randn((8192, 8192), device="cuda", dtype=torch.bfloat16)
rng = np.random.default_rng(0)


def late(value):
    """A tensor of `value` that torch has yet to fill, some 20 ms of products before it."""
    held = torch.zeros_like(value)
    y = busy
    for _ in range(15):
        y = torch.mm(y, busy)
    return held.copy_(value)


for stream in (torch.cuda.current_stream(), torch.cuda.Stream()):
    with torch.cuda.stream(stream):
        x = torch.from_numpy(rng.standard_normal((300, 2, 64)).astype(np.float32)).cuda()
        slots = torch.from_numpy(rng.permutation(400)[:300].astype(np.int32)).cuda()
        logits = torch.from_numpy(rng.standard_normal((6, 5001)).astype(np.float32)).cuda()
        state = torch.from_numpy(rng.standard_normal((6, 4, 8)).astype(np.float32)).cuda()
        want_codes, want_scales = R.quantise(x.cpu().numpy(), "i8", 32)
        want = R.values(want_codes, want_scales, "i8", 32)
        picks = R.select(logits.double().cpu().numpy(), 3, 4)
        for _ in range(3):
            codes, scales = torch.zeros((400, 2, 64), dtype=torch.uint8, device="cuda"), torch.zeros((400, 2, 2), device="cuda")
            store = ag.QuantisedRowsGPU.of_tensors(codes, scales, dev, code="i8", heads=2, dim=64, group=32)
            index = ag.UInt32ArrayGPU.of_tensor(slots, dev)
            given = late(x)
            ag.put_quantised(store, ag.RowsGPU.of_tensor(given, dev), index)
            given.zero_()
            out = late(torch.full_like(x, 7.0))  # torch's fill comes first, the rows then
            ag.take_quantised(store, index, out=ag.RowsGPU.of_tensor(out, dev))
            got = out.clone()
            assert np.array_equal(codes[slots.long()].cpu().numpy(), want_codes)
            assert (np.abs(got.cpu().numpy() - want) <= np.abs(want) * R.HALF_STEP["f32"] * 1.001).all()
            given = late(logits)
            sel = ag.select_beams(ag.RowsGPU.of_tensor(given, dev), 3, 4)
            given.zero_()
            assert np.array_equal(sel.values()[1], picks[1]) and np.array_equal(sel.values()[2], picks[2])
            parents = late(torch.from_numpy(picks[1].reshape(-1).astype(np.int32)).cuda())
            rows = ag.take_rows(ag.RowsGPU.of_tensor(state, dev), ag.UInt32ArrayGPU.of_tensor(parents, dev))[0]
            parents.fill_(99)
            assert np.array_equal(rows.values(), state.cpu().numpy()[picks[1].reshape(-1)])
            flat = late(x.reshape(-1))
            array = ag.Float32ArrayGPU.of_tensor(flat, dev)
            twice = array.add(array)
            flat.zero_()
            assert np.array_equal(twice.raw_values(), 2 * x.cpu().numpy().reshape(-1))
            total = ag.Float32ArrayGPU.of_tensor(late(torch.ones(1000, device="cuda")), dev).sum()
            assert total.raw_values()[0] == 1000.0
            assert np.array_equal(ag.Float32ArrayGPU.of_tensor(late(x.reshape(-1)), dev).raw_values(), x.cpu().numpy().reshape(-1))  # (past the small read's size)
            assert ag.UInt32ArrayGPU.of_tensor(late(slots[:5].contiguous()), dev).values() == slots[:5].tolist()
            assert np.array_equal(ag.RowsGPU.of_tensor(late(state), dev).values(), state.cpu().numpy())
            copy = ag.Float32ArrayGPU.of_tensor(late(x.reshape(-1)), dev).clone_array()
            assert np.array_equal(copy.raw_values(), x.cpu().numpy().reshape(-1))
        print("stream", stream.cuda_stream != 0, flush=True)
print("torch order OK")
