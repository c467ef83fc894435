"""Run by tests/test_gpu_rows.py in a process of its own: the row operators over torch's tensors, on torch's default stream and on another one."""
import os
import sys

import numpy as np
import torch

torch.cuda.init()
sys.path[:0] = [os.path.dirname(os.path.dirname(os.path.abspath(__file__))), os.path.dirname(os.path.abspath(__file__))]
import arrow_gpu_amd as ag  # noqa: E402
import rows_ref as R  # noqa: E402

dev = ag.GpuDevice(torch.cuda.current_device())
for stream in (torch.cuda.current_stream(), torch.cuda.Stream()):
    with torch.cuda.stream(stream):
        pipe = ag.ArrowComputePipeline(dev, "torch", hip_stream=stream.cuda_stream)
        g = torch.Generator(device="cuda").manual_seed(3)
        qkv = torch.randn((19, 8, 64), device="cuda", generator=g).to(torch.bfloat16)
        k = qkv[:, 4:6]
        codes, scales = torch.zeros((32, 2, 64), dtype=torch.uint8, device="cuda"), torch.zeros((32, 2, 2), device="cuda")
        store = ag.QuantisedRowsGPU.of_tensors(codes, scales, dev, code="i8", heads=2, dim=64, group=32)
        slots = torch.randperm(32, device="cuda", generator=g)[:19].to(torch.int32)
        out = torch.empty((19, 2, 64), device="cuda")
        ag.put_quantised_op(store, ag.RowsGPU.of_tensor(k, dev), ag.UInt32ArrayGPU.of_tensor(slots, dev), pipe)
        ag.take_quantised_op(store, ag.UInt32ArrayGPU.of_tensor(slots, dev), pipe, out=ag.RowsGPU.of_tensor(out, dev))
        x = k.float().cpu().numpy()
        c, s = R.quantise(x, "i8", 32)
        assert np.array_equal(codes.cpu().numpy()[slots.cpu().numpy()], c)
        want = R.values(c, s, "i8", 32)
        assert (np.abs(out.cpu().numpy() - want) <= np.abs(want) * R.HALF_STEP["f32"] * 1.001).all()
        lg = torch.randn((6, 501), device="cuda", generator=g).to(torch.float16)
        found = [torch.empty((2, 4), device="cuda", dtype=t) for t in (torch.float32, torch.int32, torch.int32)]
        done = torch.tensor([0b010000, 0, 0, 0, 0, 0, 0, 0], dtype=torch.uint8, device="cuda")
        sel = ag.select_beams_op(ag.RowsGPU.of_tensor(lg, dev), 3, 4, pipe, finished=ag.BooleanArrayGPU.of_tensor(done, dev, 6), out=ag.BeamSelection.of_tensors(*found, dev))
        state = torch.randn((6, 2, 5, 8), device="cuda", generator=g)
        moved = torch.zeros((8, 2, 5, 8), device="cuda")
        ag.take_rows_op(ag.RowsGPU.of_tensor(state, dev), sel.parents, pipe, out=ag.RowsGPU.of_tensor(moved, dev))
        want = R.select(lg.double().cpu().numpy(), 3, 4, finished=[0, 0, 0, 0, 1, 0])
        assert np.array_equal(found[1].cpu().numpy(), want[1]) and np.array_equal(found[2].cpu().numpy(), want[2])
        assert torch.equal(moved, state[found[1].reshape(-1).long()])
        pipe.sync()
for bad, cls in ((slots.cpu(), ag.UInt32ArrayGPU), (slots.float(), ag.UInt32ArrayGPU), (slots[::2], ag.UInt32ArrayGPU), (out.half(), ag.Float32ArrayGPU), (slots, ag.Float32ArrayGPU)):
    try:
        cls.of_tensor(bad, dev)
    except ag.ArrowErrorGPU:
        continue
    raise AssertionError((bad.dtype, bad.device, cls))
print("torch rows OK")
