"""Rows in 8 bits and attention over the hot buffer, on the GPU, against 64-bit models (tests/row_model.py).

Codes, scales and what is read back are exact.  The attention's bounds, per output element, come from what the kernel
rounds: the weights p to the 16-bit type (unit roundoff u) and the result once more (u |out|), scores and sums in 32
bits: a score is a sum of 576 products, each exact, so its error is at most 576 * 2^-23 * sum |q k| * scale (twice the
bound of an in-order sum in round-to-nearest, for the matrix unit's own order), which a weight takes over relatively;
its exponential and the division add a few units in 2^-22.  In fp16 a weight below 2^-14 loses up to 2^-25 (half the
smallest step), times the number of keys and the largest value.
"""
import numpy as np
import pytest
import torch

import row_model as rm

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
ROUND = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11}
SCALE = 192 ** -0.5


@pytest.fixture(autouse=True)
def _lib(kvops):
    kvops.clear_overflow()
    yield
    torch.cuda.synchronize()


def fmt_of(dtype, quant):
    from kv_offload_proto_amd import xds

    return xds.row_format(DT[dtype], quant=quant)


def bits_of(t):
    return t.contiguous().cpu().view(torch.int16).numpy().view(np.uint16)


def raw_values(dtype):
    def f(bits):
        return torch.from_numpy(bits.view(np.int16).copy()).view(DT[dtype]).to(torch.float64).numpy()
    return f


def latent_rows(n, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((n, rm.DIM), generator=g) * torch.exp(torch.randn((n, 1), generator=g)) * scale
    return x.to(DT[dtype])


def encoded(rows, quant):
    return torch.from_numpy(rm.encode(bits_of(rows), rows.double().numpy(), quant))


# ---- rows in 8 bits ----

@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("quant", ["latent", "row"])
@pytest.mark.parametrize("reqs,each,slots", [(1, 1, None), (1, 67, None), (3, 1, 9), (5, 13, 40)])
def test_quantize_rows(dtype, quant, reqs, each, slots):
    from kv_offload_proto_amd import xds

    fmt, n = fmt_of(dtype, quant), reqs * each
    rows = latent_rows(n, dtype, seed=each)
    rows[0, 32:64] = 0.0                                  # a group of zeros
    rows[0, 64] = 0.0
    rows[-1, 1] = 448.0 * 1.0009765625                    # the groups' largest beside a power of two times 448
    rows[-1, 33] = 448.0 if dtype == "fp16" else 449.0
    want = encoded(rows, quant)
    total = n if slots is None else reqs * slots
    hot = torch.full((total, fmt.row_bytes), 0xA5, dtype=torch.uint8)
    rng = np.random.default_rng(n)
    if slots is None:
        at, expect = None, want
    else:
        at = np.stack([rng.permutation(slots)[:each] for _ in range(reqs)]).astype(np.int32)
        at[0, 0] = -1 if each > 1 else at[0, 0]
        expect = hot.clone()
        for i, s in enumerate(at.reshape(-1)):
            if s >= 0:
                expect[(i // each) * slots + int(s)] = want[i]
        at = torch.from_numpy(at).cuda()
    dev = hot.cuda()
    xds.quantize_rows(fmt, rows.cuda(), dev, at, slots or 0)
    assert torch.equal(dev.cpu(), expect)


@pytest.mark.parametrize("quant", ["latent", "row"])
def test_quantize_rows_special_values(quant):
    """NaN, infinities, the smallest and the largest values of bf16; every 16-bit pattern once."""
    from kv_offload_proto_amd import xds

    fmt = fmt_of("bf16", quant)
    bits = np.arange(1 << 16, dtype=np.uint16)
    bits = np.concatenate([bits, np.zeros(-len(bits) % rm.DIM, np.uint16)]).reshape(-1, rm.DIM)
    mixed = np.random.default_rng(1).permutation(bits.reshape(-1)).reshape(bits.shape)
    bits = np.concatenate([bits, mixed])
    values = raw_values("bf16")(bits)
    want = rm.encode(bits, values, quant)
    rows = torch.from_numpy(bits.view(np.int16)).view(torch.bfloat16).cuda()
    hot = torch.empty((rows.shape[0], fmt.row_bytes), dtype=torch.uint8, device="cuda")
    xds.quantize_rows(fmt, rows, hot)
    got = hot.cpu().numpy()
    d = rm.CODES[quant]
    nan = np.isnan(values[:, :d])
    assert np.array_equal(got[:, :d][nan] & 127, np.full(nan.sum(), 127))
    assert np.array_equal(got[:, :d][~nan], want[:, :d][~nan])
    assert np.array_equal(got[:, d:], want[:, d:])


def test_quantize_rows_of_a_strided_tensor():
    from kv_offload_proto_amd import xds

    fmt = fmt_of("bf16", "row")
    wide = torch.randn((9, 640), dtype=torch.float32).to(torch.bfloat16)
    want = encoded(wide[:, 32:608], "row")
    for view in (wide.cuda()[:, 32:608], wide.cuda()[:, 32:608].reshape(3, 3, rm.DIM)):
        hot = torch.zeros((9, fmt.row_bytes), dtype=torch.uint8, device="cuda")
        xds.quantize_rows(fmt, view, hot)
        assert torch.equal(hot.cpu(), want)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("quant", ["latent", "row"])
@pytest.mark.parametrize("out", ["bf16", "fp16", "fp32"])
def test_dequantize_rows(dtype, quant, out):
    """Every code under scales from the smallest to the largest, holes, rows out of order."""
    from kv_offload_proto_amd import xds

    fmt, n = fmt_of(dtype, quant), 77
    rng = np.random.default_rng(n)
    rec = rm.encode(bits_of(latent_rows(n, dtype, 5)), latent_rows(n, dtype, 5).double().numpy(), quant)
    d = rm.CODES[quant]
    rec[:40, :d] = (np.arange(40 * d) % 256).reshape(40, d)
    end = d + 2 * (rm.DIM - d)
    rec[:40, end:end + d // 32] = rng.integers(0, 248, (40, d // 32))
    rec[0, end:end + d // 32] = np.arange(d // 32)
    slots = rng.permutation(n)[:70].reshape(7, 10).astype(np.int32)
    slots[rng.random(slots.shape) < 0.2] = -1
    values = rm.decode(rec, raw_values(dtype), quant)
    kind = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}[out]
    # a code's value has 4 significant bits: exact in 32 bits, so one rounding
    want = torch.from_numpy(values).to(torch.float32).to(kind)
    hot = torch.from_numpy(rec).cuda()
    every = xds.dequantize_rows(fmt, hot, dtype=kind)
    assert torch.equal(every.cpu().nan_to_num(1.0, posinf=2.0, neginf=3.0), want.nan_to_num(1.0, posinf=2.0, neginf=3.0))
    got = xds.dequantize_rows(fmt, hot, torch.from_numpy(slots).cuda(), 0, dtype=kind).cpu()
    pick = torch.from_numpy(slots.reshape(-1).astype(np.int64))
    part = torch.where((pick >= 0)[:, None], want[pick.clamp(min=0)].float(), torch.zeros(())).to(kind)
    assert torch.equal(got.nan_to_num(1.0, posinf=2.0, neginf=3.0), part.nan_to_num(1.0, posinf=2.0, neginf=3.0))


def test_round_trip_is_within_half_a_step():
    from kv_offload_proto_amd import xds

    rows = latent_rows(129, "bf16", 9)
    fmt = fmt_of("bf16", "row")
    hot = torch.empty((129, fmt.row_bytes), dtype=torch.uint8, device="cuda")
    xds.quantize_rows(fmt, rows.cuda(), hot)
    back = xds.dequantize_rows(fmt, hot, dtype=torch.float32).cpu()
    x = rows.float()
    top = x.abs().reshape(129, 18, 32).amax(2, keepdim=True).expand(-1, -1, 32).reshape(129, 576)
    # 4 significant bits: half a step is 2^-4 of the value; below the smallest normal code, half of 2^-9 of a scale
    # that is under top / 224
    assert bool(((back - x).abs() <= torch.maximum(x.abs() * 2.0 ** -4, top / 224 * 2.0 ** -10)).all())


# ---- attention ----

def problem(reqs, tokens, heads, top_k, slots, dtype, quant, tree, holes=0.0, seed=0, q_scale=1.0):
    rng = np.random.default_rng(seed + 1000 * tokens + top_k)
    stride = -(-slots // 16) * 16 + (tokens if tree else 0)
    rows = latent_rows(reqs * stride, dtype, seed + 1)
    p = dict(fmt=fmt_of(dtype, quant), dtype=dtype, quant=quant, stride=stride, hot=encoded(rows, quant))
    g = torch.Generator().manual_seed(seed + 2)
    p["q"] = (torch.randn((reqs, tokens, heads, rm.DIM), generator=g) * q_scale).to(DT[dtype])
    at = np.stack([rng.permutation(slots)[:top_k] for _ in range(reqs)]).astype(np.int32).reshape(reqs, top_k)
    at[rng.random(at.shape) < holes] = -1
    p["slots"] = at
    p["draft_slots"] = p["tree_mask"] = None
    if tree:
        p["draft_slots"] = np.tile(np.arange(stride - tokens, stride, dtype=np.int32), (reqs, 1))
        mask = np.zeros((reqs, tokens), np.uint64)
        for b in range(reqs):
            for t in range(tokens):
                up = mask[b, t - rng.integers(1, min(t, 4) + 1)] if t else np.uint64(0)
                mask[b, t] = up | np.uint64(1 << t)
        p["tree_mask"] = mask
    return p


def dev(a):
    if a is None or isinstance(a, torch.Tensor):
        return a if a is None else a.cuda()
    return torch.from_numpy(np.ascontiguousarray(a.view(np.int64) if a.dtype == np.uint64 else a)).cuda()


def run(p, **over):
    from kv_offload_proto_amd import xds

    v = {k: dev(over.get(k, p[k])) for k in ("q", "hot", "slots", "draft_slots", "tree_mask")}
    return xds.tree_attention(p["fmt"], v["q"], v["hot"], v["slots"], over.get("scale", SCALE), p["stride"],
                              draft_slots=v["draft_slots"], tree_mask=v["tree_mask"], out=over.get("out"),
                              lse=over.get("lse"))


def model(p, scale=SCALE):
    hot = p["hot"].numpy()
    keys = rm.keys_of(p["slots"], p["draft_slots"], p["tree_mask"], p["stride"], hot.shape[0])
    return rm.attention(p["q"].double().numpy(),
                        lambda rows: rm.decode(hot[rows], raw_values(p["dtype"]), p["quant"]), keys, scale)


def check(p, out, lse, scale=SCALE, expected=None):
    want, want_lse, weighted, size = model(p, scale) if expected is None else expected
    got, got_lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
    u = ROUND[p["dtype"]]
    score = 576 * 2.0 ** -23 * size                        # absolute error of a score (natural units)
    keys = p["slots"].shape[1] + 64
    lost = keys * 2.0 ** -25 * np.abs(rm.decode(p["hot"].numpy(), raw_values(p["dtype"]), p["quant"])[:, :512]).max()
    tol = u * np.abs(want) + (u + 2 * score + 2.0 ** -18)[..., None] * weighted + (lost if p["dtype"] == "fp16" else 0)
    assert np.isfinite(got).all()
    worst = np.max(np.abs(got - want) - 1.01 * tol - 1e-30)
    assert worst <= 0, worst
    empty = np.isneginf(want_lse)
    assert np.array_equal(np.isneginf(got_lse), empty) and not got[empty].any()
    d = np.abs(got_lse - want_lse)[~empty]
    assert (d <= (score + 2.0 ** -20 * (1 + np.abs(want_lse)))[~empty]).all(), d.max()


CASES = [
    # requests, tokens, heads, topK, slots, dtype, quant, tree, holes
    (1, 1, 1, 1, 1, "bf16", "none", False, 0),
    (1, 1, 1, 1, 2, "fp16", "row", True, 0),
    (8, 1, 16, 64, 64, "fp16", "none", False, 0),
    (3, 1, 16, 65, 70, "bf16", "latent", False, 0.1),
    (2, 1, 128, 300, 512, "bf16", "row", False, 0),
    (2, 1, 128, 257, 300, "bf16", "none", True, 0),
    (2, 3, 5, 63, 80, "fp16", "latent", True, 0.3),
    (1, 7, 20, 333, 1000, "bf16", "row", True, 0.05),
    (2, 64, 3, 40, 50, "bf16", "none", True, 0.5),
    (1, 64, 1, 1, 3, "fp16", "row", True, 0),
    (1, 4, 33, 1000, 1300, "fp16", "none", True, 0),
    (1, 9, 128, 130, 200, "fp16", "latent", True, 0),
    (1, 1, 8, 2500, 4000, "bf16", "none", False, 0.02),
    (1, 2, 64, 4100, 4300, "fp16", "row", True, 0),
    (65, 1, 4, 5, 9, "bf16", "row", True, 0.2),
    (1, 1, 200, 31, 40, "bf16", "none", True, 0),
]


@pytest.mark.parametrize("reqs,tokens,heads,top_k,slots,dtype,quant,tree,holes", CASES)
def test_tree_attention(reqs, tokens, heads, top_k, slots, dtype, quant, tree, holes):
    p = problem(reqs, tokens, heads, top_k, slots, dtype, quant, tree, holes)
    out, lse = run(p)
    check(p, out, lse)
    again, lse2 = run(p)
    assert torch.equal(out, again) and torch.equal(lse, lse2)   # nothing depends on an order


@pytest.mark.parametrize("dtype,quant", [("bf16", "none"), ("fp16", "row"), ("fp16", "none")])
@pytest.mark.parametrize("q_scale", [30.0, 0.0])
def test_scores_far_apart_and_all_alike(dtype, quant, q_scale):
    """A maximum that keeps rising from tile to tile, by hundreds; and weights that are all one."""
    p = problem(2, 2, 16, 700, 900, dtype, quant, True, q_scale=q_scale)
    check(p, *run(p))


def test_rising_scores():
    """Keys in ascending order of their score: every tile raises the maximum."""
    p = problem(1, 1, 40, 640, 640, "bf16", "none", False)
    q = p["q"][0, 0, 0].double().numpy()
    p["q"][0, 0, :] = p["q"][0, 0, 0]
    rows = rm.decode(p["hot"].numpy(), raw_values("bf16"), "none")
    p["slots"] = np.argsort(rows[:640] @ q).astype(np.int32)[None]
    check(p, *run(p))
    p["slots"] = np.ascontiguousarray(p["slots"][:, ::-1])
    check(p, *run(p))


@pytest.mark.parametrize("heads", [4, 128])
@pytest.mark.parametrize("dtype,quant", [("bf16", "none"), ("fp16", "latent"), ("bf16", "row")])
def test_unseen_rows_have_no_effect(heads, dtype, quant):
    """NaN, infinities and the type's largest values in every row that a query does not see."""
    p = problem(3, 6, heads, 90, 200, dtype, quant, True, holes=0.2)
    p["slots"][1] = -1                                      # a request with no selection
    p["tree_mask"][1, 2] = 0                                # ... one of whose tokens sees nothing at all
    p["draft_slots"][2, 4] = -1                             # a token without a row
    p["tree_mask"][0, :] &= np.uint64(~(1 << 3) & (2 ** 64 - 1))
    p["tree_mask"][0, 3] |= np.uint64(1 << 3)               # token 3 of request 0 is seen by itself alone
    clean = run(p)
    check(p, *clean)
    used = set()
    for b, (rows, seen) in enumerate(rm.keys_of(p["slots"], p["draft_slots"], p["tree_mask"], p["stride"],
                                                p["hot"].shape[0])):
        used |= {int(r) for r, s in zip(rows, seen.T) if s.any()}
    hot = p["hot"].clone()
    hot[[r for r in range(hot.shape[0]) if r not in used]] = 0xFF    # NaN in every form
    for got, want in zip(run(p, hot=hot), clean):
        assert torch.equal(got, want)
    # token 3 of request 0 sees its own row, the others must not
    for byte in (0xFF, 0x7F):
        hot[p["draft_slots"][0, 3]] = byte
        out, lse = run(p, hot=hot)
        keep = torch.ones((3, 6), dtype=torch.bool)
        keep[0, 3] = False
        assert torch.equal(out[keep.cuda()], clean[0][keep.cuda()])
        assert torch.equal(lse[keep.cuda()], clean[1][keep.cuda()])
        if byte == 0xFF:
            assert bool(out[0, 3].isnan().all()) and bool(lse[0, 3].isnan().all())
    if quant == "none":
        inf = torch.tensor([0x7F80 if dtype == "bf16" else 0x7C00], dtype=torch.int16).view(torch.uint8)
        hot[p["draft_slots"][0, 3]] = inf.repeat(576)
        out, lse = run(p, hot=hot)
        assert torch.equal(out[keep.cuda()], clean[0][keep.cuda()])


def test_no_keys():
    p = problem(2, 3, 20, 70, 80, "bf16", "row", True)
    p["slots"][:] = -1
    p["draft_slots"][:] = -1
    out, lse = run(p)
    assert not bool(out.any()) and bool(torch.isneginf(lse).all())
    p["slots"] = p["slots"][:, :0]
    p["draft_slots"] = p["tree_mask"] = None
    out, lse = run(p)
    assert not bool(out.any()) and bool(torch.isneginf(lse).all())


def test_slots_that_repeat_count_twice():
    p = problem(1, 1, 16, 50, 60, "fp16", "none", False)
    p["slots"][0, 10:30] = p["slots"][0, 0]
    check(p, *run(p))


def test_chain_is_the_default_mask():
    p = problem(2, 5, 16, 33, 40, "bf16", "none", True)
    p["tree_mask"] = None
    out, lse = run(p)
    check(p, out, lse)
    chain = np.tile(np.array([(2 << t) - 1 for t in range(5)], np.uint64), (2, 1))
    again, _ = run(p, tree_mask=chain)
    assert torch.equal(out, again)


def test_negative_scale():
    p = problem(1, 1, 16, 100, 120, "bf16", "none", False)
    out, lse = run(p, scale=-0.05)
    check(p, out, lse, scale=-0.05)


def test_strided_queries():
    """Heads before tokens, and queries inside a wider projection."""
    p = problem(2, 3, 10, 70, 90, "bf16", "latent", True)
    want, want_lse = run(p)
    swapped = p["q"].transpose(1, 2).contiguous().cuda().transpose(1, 2)
    wide = torch.full((2, 3, 10, 640), float("nan"), dtype=torch.bfloat16, device="cuda")
    wide[..., 64:] = p["q"].cuda()
    for q in (swapped, wide[..., 64:]):
        assert not q.is_contiguous()
        out, lse = run(p, q=q)
        assert torch.equal(out, want) and torch.equal(lse, want_lse)


def test_rows_past_four_gibibytes():
    """Slots and requests whose bytes lie behind 2^32, in one request and between them."""
    from kv_offload_proto_amd import xds

    fmt = fmt_of("bf16", "none")
    p = problem(2, 1, 16, 70, 80, "bf16", "none", False)
    stride, shift = 4_000_000, 3_900_000                     # 4.6 GB a request
    hot = torch.empty((2 * stride, fmt.row_bytes), dtype=torch.uint8, device="cuda")
    for b in range(2):
        hot[b * stride + shift:b * stride + shift + 80] = p["hot"][b * p["stride"]:b * p["stride"] + 80].cuda()
    slots = torch.from_numpy(p["slots"] + shift).cuda()
    want, want_lse = run(p)
    out, lse = xds.tree_attention(fmt, p["q"].cuda(), hot, slots, SCALE, stride)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    del hot
    fmt8 = fmt_of("bf16", "row")
    hot = torch.empty((7_000_000, fmt8.row_bytes), dtype=torch.uint8, device="cuda")
    rows = latent_rows(4, "bf16", 3).cuda()
    at = torch.tensor([[6_999_990, 6_999_999], [3, 6_900_000]], dtype=torch.int32, device="cuda")
    xds.quantize_rows(fmt8, rows, hot, at)
    assert torch.equal(hot[at.reshape(-1).long()].cpu(), encoded(rows.cpu(), "row"))
    got = xds.dequantize_rows(fmt8, hot, at)
    assert torch.equal(got, xds.dequantize_rows(fmt8, hot[at.reshape(-1).long()]))


def test_slot_past_the_buffer_is_told(kvops):
    from kv_offload_proto_amd import xds

    p = problem(2, 1, 16, 40, 64, "bf16", "row", False)
    p["slots"][1, 7] = 64
    want = run(p, slots=np.where(p["slots"] == 64, -1, p["slots"]))
    assert kvops.read_overflow() == 0
    got = run(p)
    assert kvops.read_overflow() == 0x524F57
    assert torch.equal(got[0], want[0])
    kvops.clear_overflow()
    hot, at = p["hot"].cuda(), torch.tensor([[3, 200]], dtype=torch.int32, device="cuda")
    rows = latent_rows(2, "bf16", 3).cuda()
    xds.quantize_rows(p["fmt"], rows, hot, at)
    assert kvops.read_overflow() == 0x524F57
    expect = p["hot"].clone()
    expect[3] = encoded(rows.cpu(), "row")[0]
    assert torch.equal(hot.cpu(), expect)
    kvops.clear_overflow()
    back = xds.dequantize_rows(p["fmt"], hot, at)
    assert kvops.read_overflow() == 0x524F57 and not bool(back[1].any()) and bool(back[0].any())
    kvops.clear_overflow()


def test_two_streams_at_once():
    """Calls of one shape on two streams: neither sees what the other keeps."""
    a, b = (problem(2, 2, 32, 1500, 1600, "bf16", "none", True, seed=s) for s in (1, 2))
    want = [run(a), run(b)]
    args = [{k: dev(p[k]) for k in ("q", "hot", "slots", "draft_slots", "tree_mask")} for p in (a, b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(5):
        for i, (p, st) in enumerate(zip((a, b), streams)):
            with torch.cuda.stream(st):
                got[i].append(run(p, **args[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for out, lse in got[i]:
            assert torch.equal(out, want[i][0]) and torch.equal(lse, want[i][1])


def test_explicit_stream():
    from kv_offload_proto_amd import xds

    fmt, st = fmt_of("bf16", "row"), torch.cuda.Stream()
    rows = latent_rows(33, "bf16", 3).cuda()
    hot = torch.zeros((33, fmt.row_bytes), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    xds.quantize_rows(fmt, rows, hot, stream=st)
    out = torch.empty((33, rm.DIM), dtype=torch.bfloat16, device="cuda")
    xds.dequantize_rows(fmt, hot, out=out, stream=st.cuda_stream)
    st.synchronize()
    assert torch.equal(hot.cpu(), encoded(rows.cpu(), "row"))
    assert torch.equal(out, xds.dequantize_rows(fmt, hot))


def test_refusals():
    from kv_offload_proto_amd import xds

    p = problem(2, 2, 4, 8, 16, "bf16", "row", True)
    fmt, v = p["fmt"], {k: dev(p[k]) for k in ("q", "hot", "slots", "draft_slots", "tree_mask")}

    def attend(fmt=fmt, scale=SCALE, stride=p["stride"], **over):
        w = {**v, **over}
        return xds.tree_attention(fmt, w["q"], w["hot"], w["slots"], scale, stride, draft_slots=w["draft_slots"],
                                  tree_mask=w["tree_mask"], out=w.get("out"), lse=w.get("lse"))

    attend()
    bad = [
        dict(q=v["q"].half()), dict(q=v["q"].cpu()), dict(q=v["q"][..., :512]), dict(q=v["q"][0]),
        dict(q=torch.zeros((2, 2, 4, 1152), dtype=torch.bfloat16, device="cuda")[..., ::2]),
        dict(q=torch.zeros((2, 2, 4, 580), dtype=torch.bfloat16, device="cuda")[..., :576]),
        dict(hot=v["hot"].cpu()), dict(hot=v["hot"].reshape(-1)[:-1]), dict(hot=v["hot"][:, ::2]),
        dict(slots=v["slots"].long()), dict(slots=v["slots"][:1]), dict(slots=v["slots"].cpu()),
        dict(slots=v["slots"][:, ::2]), dict(draft_slots=v["draft_slots"][:, :1]), dict(draft_slots=v["draft_slots"].long()),
        dict(tree_mask=v["tree_mask"].int()), dict(tree_mask=v["tree_mask"][:, :1]), dict(draft_slots=None),
        dict(out=torch.empty((2, 2, 4, 512), device="cuda")), dict(out=torch.empty((2, 2, 4, 576), dtype=torch.bfloat16, device="cuda")),
        dict(lse=torch.empty((2, 2, 5), device="cuda")), dict(stride=-1),
    ]
    for over in bad:
        with pytest.raises(ValueError):
            attend(**over)
    with pytest.raises(RuntimeError, match="draft must be <= 64"):
        attend(q=torch.zeros((2, 65, 4, 576), dtype=torch.bfloat16, device="cuda"), draft_slots=None, tree_mask=None)
    with pytest.raises(RuntimeError, match="heads must be <= 1024"):
        attend(q=torch.zeros((2, 1, 1025, 576), dtype=torch.bfloat16, device="cuda"), draft_slots=None, tree_mask=None)
    with pytest.raises(RuntimeError, match="16-byte aligned"):
        attend(q=torch.zeros(2 * 2 * 4 * 576 + 4, dtype=torch.bfloat16, device="cuda")[4:].reshape(2, 2, 4, 576))

    rows = torch.zeros((4, 576), dtype=torch.bfloat16, device="cuda")
    for args in [(xds.row_format(torch.bfloat16), rows, v["hot"]), (fmt, rows.half(), v["hot"]), (fmt, rows[:, :512], v["hot"]),
                 (fmt, torch.zeros((4, 580), dtype=torch.bfloat16, device="cuda")[:, :576], v["hot"]), (fmt, rows.cpu(), v["hot"]), (fmt, rows, v["hot"][:2].contiguous()), (fmt, rows, v["hot"], v["slots"]),
                 (fmt, rows, v["hot"], torch.zeros((2, 2), device="cuda", dtype=torch.int64))]:
        with pytest.raises(ValueError):
            xds.quantize_rows(*args)
    for kw in [dict(out=torch.empty((4, 512), device="cuda")), dict(out=torch.empty((4, 576), dtype=torch.float64, device="cuda")),
               dict(out=torch.empty((10 ** 4, 576), device="cuda")), dict(out=torch.empty((4, 576), device="cuda"), dtype=torch.bfloat16)]:
        with pytest.raises(ValueError):
            xds.dequantize_rows(fmt, v["hot"], **kw)
    with pytest.raises(ValueError):
        xds.dequantize_rows(xds.row_format(torch.bfloat16), v["hot"])


def test_empty_calls():
    """No requests, no tokens, no rows: nothing to do and no error."""
    from kv_offload_proto_amd import xds

    fmt = fmt_of("bf16", "row")
    hot = torch.zeros((4, fmt.row_bytes), dtype=torch.uint8, device="cuda")
    for shape in [(0, 1, 4), (2, 0, 4), (2, 1, 0)]:
        q = torch.zeros(shape + (576,), dtype=torch.bfloat16, device="cuda")
        out, lse = xds.tree_attention(fmt, q, hot, torch.zeros((2, 3), dtype=torch.int32, device="cuda"), 1.0)
        assert out.shape == shape + (512,) and lse.shape == shape
    xds.quantize_rows(fmt, torch.zeros((0, 576), dtype=torch.bfloat16, device="cuda"), hot)
    assert xds.dequantize_rows(fmt, hot, torch.zeros((3, 0), dtype=torch.int32, device="cuda")).shape == (0, 576)
