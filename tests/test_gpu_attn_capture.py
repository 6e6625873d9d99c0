"""What ends while the library's stream is captured (sllm_gfx950_attn.h), on the GPU:
the capture goes on, and what it recorded is right on every replay."""
import numpy as np
import pytest
import torch

import attn_oracle as ora

pytestmark = pytest.mark.gpu


def test_ends_in_a_capture(amd, dev):
    torch.cuda.init()
    stream = torch.cuda.ExternalStream(amd.lib().sllm_gfx950_stream())
    heads, kv, d = 4, 2, 64
    c, other = (amd.PagedCache(dev, 1, kv, d, 16, 60, "float16") for _ in range(2))
    s = c.new()
    b = c.batch([s], [50], heads)
    gone = [c.batch([c.new()], [10 * (i + 1)], heads) for i in range(6)]
    plan = amd.PromptAttention(dev, "float16", heads, kv, d, [9, 40])
    g = torch.Generator()
    g.manual_seed(3)
    x = [dev.put(ora.bits(torch.randn(50, h, d, generator=g).half())) for h in (heads, kv, kv)]
    out = dev.alloc(50 * heads * d * 2)
    b.store(0, x[1].ptr, x[2].ptr)
    b.attend(0, x[0].ptr, out.ptr, 0.125)
    dev.sync()
    want = out.download(np.int16, 50 * heads * d)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
        b.store(0, x[1].ptr, x[2].ptr)
        for y in gone:
            y.close()
        plan.close()
        other.close()
        b.attend(0, x[0].ptr, out.ptr, 0.125)
    for turn in range(3):
        out.upload(np.zeros(want.size, np.int16))
        with torch.cuda.stream(stream):
            graph.replay()
        dev.sync()
        assert np.array_equal(out.download(np.int16, want.size), want), turn
        if turn == 0:
            again = c.fork(s, 37, 1)                     # now what ended is freed
            c.free(again)
        b.attend(0, x[0].ptr, out.ptr, 0.125)
        dev.sync()
        assert np.array_equal(out.download(np.int16, want.size), want), turn
    b.close()
    c.close()
    for y in x + [out]:
        y.free()
