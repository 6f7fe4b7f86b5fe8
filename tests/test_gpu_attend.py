"""The operators on the cache rows where a decode loop has them: recorded into
a graph, and behind the SIEVE update and the imports."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from test_gpu_attention import check, dev, problem, run

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(autouse=True)
def _lib(kvops):
    yield
    torch.cuda.synchronize()


# requests, tokens, heads, topK, slots, dtype, quant, tree: keys of a query in several workgroups, for the kernels of 16
# and of more queries a workgroup, and in one
GRAPHS = [
    (1, 1, 8, 2500, 4000, "bf16", "none", False),
    (1, 9, 128, 1030, 1200, "fp16", "row", True),
    (8, 1, 16, 64, 64, "bf16", "latent", False),
]


@pytest.mark.parametrize("reqs,tokens,heads,top_k,slots,dtype,quant,tree", GRAPHS)
def test_replays_match_eager_calls(reqs, tokens, heads, top_k, slots, dtype, quant, tree):
    """quantize_rows and tree_attention captured; every replay with new inputs, eager work and syncs between."""
    from kv_offload_proto_amd import xds

    problems = [problem(reqs, tokens, heads, top_k, slots, dtype, quant, tree, seed=s) for s in range(4)]
    fmt, stride = problems[0]["fmt"], problems[0]["stride"]
    v = {k: dev(problems[0][k]) for k in ("q", "hot", "slots", "draft_slots", "tree_mask")}
    out = torch.empty((reqs, tokens, heads, 512), dtype=fmt.dtype, device="cuda")
    lse = torch.empty((reqs, tokens, heads), device="cuda")
    new = torch.randn((reqs * tokens, 576), device="cuda").to(fmt.dtype)

    def step():
        if tree and quant != "none":
            xds.quantize_rows(fmt, new, v["hot"], v["draft_slots"], stride)
        return run(problems[0], **v, out=out, lse=lse)

    side = torch.cuda.Stream()
    xds.reserve_attention(fmt, reqs, tokens, heads, top_k, drafted=tree, stream=side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    for p in problems[1:] + problems[:1]:
        for k in v:
            if v[k] is not None:
                v[k].copy_(dev(p[k]))
        new.normal_()
        hot = v["hot"].clone()
        out.fill_(float("nan"))
        lse.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        got, got_lse, after = out.clone(), lse.clone(), v["hot"].clone()
        v["hot"].copy_(hot)
        step()
        assert torch.equal(got, out) and torch.equal(got_lse, lse) and torch.equal(after, v["hot"])
        assert bool(torch.isfinite(got).all())


def test_capture_without_reserve_is_refused():
    p = problem(1, 1, 8, 2500, 4000, "bf16", "none", False)
    v = {k: dev(p[k]) for k in ("q", "hot", "slots", "draft_slots", "tree_mask")}
    out = torch.empty((1, 1, 8, 512), dtype=torch.bfloat16, device="cuda")
    lse = torch.empty((1, 1, 8), device="cuda")
    side = torch.cuda.Stream()
    mark = torch.zeros(1, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        with pytest.raises(RuntimeError, match="call reserve_attention for the stream before capturing"):
            run(p, **v, out=out, lse=lse)
        mark.add_(1)
    graph.replay()
    torch.cuda.synchronize()
    assert mark.item() == 1.0


def test_reserve_grows_once(kvops):
    from kv_offload_proto_amd import xds

    st = torch.cuda.Stream()
    fmt = xds.row_format(torch.bfloat16)
    assert kvops.scratch_bytes(st.cuda_stream) == 0
    xds.reserve_attention(fmt, 8, 1, 16, 64, stream=st)          # one workgroup a query: nothing to keep
    assert kvops.scratch_bytes(st.cuda_stream) == 0
    xds.reserve_attention(fmt, 1, 1, 16, 8192, stream=st)
    size = kvops.scratch_bytes(st.cuda_stream)
    assert size >= 2 * 16 * 514 * 4
    xds.reserve_attention(fmt, 1, 1, 16, 8192, stream=st)
    xds.reserve_attention(fmt, 1, 1, 4, 8192, stream=st)
    assert kvops.scratch_bytes(st.cuda_stream) == size
    with pytest.raises(RuntimeError, match="draft must be <= 64"):
        xds.reserve_attention(fmt, 1, 65, 16, 8192, stream=st)
    with pytest.raises(RuntimeError, match="heads must be <= 1024"):
        xds.reserve_attention(fmt, 1, 1, 1025, 8192, stream=st)
    with pytest.raises(ValueError):
        xds.reserve_attention(fmt, 1, 1, -1, 8192, stream=st)


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), float("-inf")])
def test_scale_that_is_not_finite_is_refused(scale):
    with pytest.raises(RuntimeError, match="softmax_scale must be finite"):
        run(problem(1, 1, 2, 4, 8, "bf16", "row", False), scale=scale)


@pytest.mark.parametrize("heads,dtype,quant", [(3, "bf16", "none"), (150, "fp16", "row")])
def test_scale_of_zero_weighs_all_alike(heads, dtype, quant):
    p = problem(2, 3, heads, 70, 90, dtype, quant, True, holes=0.2)
    check(p, *run(p, scale=0.0), scale=0.0)


@pytest.mark.parametrize("dtype", [torch.float64, torch.int16])
def test_values_of_another_type_are_refused(dtype):
    from kv_offload_proto_amd import xds

    fmt = xds.row_format(torch.bfloat16, quant="row")
    with pytest.raises(ValueError, match="dtype must be"):
        xds.dequantize_rows(fmt, torch.zeros((4, fmt.row_bytes), dtype=torch.uint8, device="cuda"), dtype=dtype)


@pytest.mark.parametrize("flags", [
    [],
    ["--quant", "latent", "--dtype", "fp16", "--draft", "1", "--heads", "5", "--topk", "33"],
    ["--quant", "none", "--draft", "9", "--heads", "32", "--prefill", "700", "--topk", "150",
     "--device-buffer-size", "320", "--req-num", "3", "--layers", "3", "--steps", "6", "--node-num", "3"],
    ["--device-buffer-size", "64", "--dtype", "fp16"],           # slots taken again within one update
])
def test_decode_steps_that_attend(flags):
    """Every output of the example against the formula in 64 bits, which it does by itself."""
    cmd = [sys.executable, "-u", "-m", "kv_offload_proto_amd.xds.xds_attend"] + flags
    done = subprocess.run(cmd, cwd=ROOT, capture_output=True, text=True, timeout=110)
    text = done.stdout
    print(text[-3000:], done.stderr[-2000:], flush=True)
    assert done.returncode == 0 and "[xds][ERROR]" not in text and "[xds] all done" in text
    assert text.count("[xds] step ") == (6 if "--steps" in flags else 10)
    misses = [int(line.split("miss=")[1].split()[0]) for line in text.splitlines() if "miss=" in line]
    assert any(misses)
    assert np.isfinite(float(text.split("largest error ")[1].split()[0]))
