"""The 8-bit row model and the row formats, without a GPU."""
import numpy as np
import pytest
import torch

import row_model as rm


def test_codes_are_e4m3():
    """The model's codes against torch's conversion, over every code, the middles between codes, and beside them."""
    v = rm.CODE_VALUES[:127]
    x = np.concatenate([v, (v[:-1] + v[1:]) / 2, np.nextafter((v[:-1] + v[1:]) / 2, 0), np.nextafter((v[:-1] + v[1:]) / 2, 500)])
    x = np.concatenate([x, -x]).astype(np.float32)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(rm.e4m3(x.astype(np.float64)), want)
    back = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(back, rm.CODE_VALUES, equal_nan=True)


@pytest.mark.parametrize("quant", ["latent", "row"])
def test_model_scale_is_the_smallest_that_fits(quant):
    rows = (torch.randn((9, 576), generator=torch.Generator().manual_seed(1)) * 3).to(torch.bfloat16)
    rec = rm.encode(rows.view(torch.int16).numpy().view(np.uint16), rows.double().numpy(), quant)
    d = rm.CODES[quant]
    end = d + 2 * (576 - d)
    scale = 2.0 ** (rec[:, end:end + d // 32].astype(float) - 127)
    top = rows.double().abs()[:, :d].reshape(9, -1, 32).amax(2).numpy()
    assert (top <= 448 * scale).all() and (top > 224 * scale).all()


def test_row_formats():
    from kv_offload_proto_amd.xds import RowFormat, configs, row_format

    assert [row_format(torch.float16, quant=k).row_bytes for k in ("none", "latent", "row")] == [1152, 768, 640]
    assert row_format(torch.float16).row_bytes == configs.row_bytes_of()
    assert row_format(torch.bfloat16, quant="row") is row_format(torch.bfloat16, quant="row")
    assert all(row_format(torch.bfloat16, quant=k).row_bytes % 128 == 0 for k in ("none", "latent", "row"))
    for kw in (dict(dtype=torch.float32), dict(kv_lora_rank=511), dict(qk_rope=0), dict(quant="int8")):
        with pytest.raises(ValueError):
            RowFormat(**kw)


def test_calls_refuse_host_tensors():
    from kv_offload_proto_amd import xds

    fmt = xds.row_format(torch.bfloat16, quant="row")
    hot = torch.zeros((4, fmt.row_bytes), dtype=torch.uint8)
    with pytest.raises(ValueError, match="on the GPU"):
        xds.quantize_rows(fmt, torch.zeros((1, 576), dtype=torch.bfloat16), hot)
    with pytest.raises(ValueError, match="on the GPU"):
        xds.dequantize_rows(fmt, hot)
    with pytest.raises(ValueError, match="on the GPU"):
        xds.tree_attention(fmt, torch.zeros((1, 1, 1, 576), dtype=torch.bfloat16), hot,
                           torch.zeros((1, 1), dtype=torch.int32), 1.0)


def test_header_declares_what_the_library_exports():
    import ctypes
    import os
    import re

    import kv_offload_proto_amd  # noqa: F401
    from kv_offload_proto_amd.kvops_ext import lib_path

    here = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(here, "include", "kvx", "kvx_attn.h")).read(), flags=re.S)
    names = set(re.findall(r"\b(kvx_\w+)\s*\(", text))
    lib = ctypes.CDLL(lib_path())
    assert names and all(hasattr(lib, n) for n in names)
