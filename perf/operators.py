"""The quantised cache rows and the attention over the hot buffer, as cases to be timed.

A cache row is one latent row, (512 + 64) 16-bit values: 512 that serve as keys and values of every query head, and 64
rotary ones that serve as keys only.  A decode server has this package

* write rows in 8 bits (``quantize_rows``): each new token's row of every request to its place in the hot buffer, and a
  prompt's rows of every layer, before they are exported to the host segments (a miss then moves 640 bytes over the
  host link instead of 1152);
* read selected rows back in 16 bits (``dequantize_rows``), for a program that runs its own attention on them;
* attend (``tree_attention``): the queries of each request's drafted tokens (one, where nothing is drafted) over the
  slots that its topK selection named and over the drafted tokens' own rows, each drafted token seeing its ancestors.

The plain forms are elementary torch operations in 32 bits; ``exact`` goes by the definitions in 64 bits.

A row in 8 bits holds groups of 32 values as e4m3 codes with one power-of-two scale, the smallest for which the
group's largest finite magnitude is at most 448 codes:

* ``quant="row"``:    576 codes, 18 scale exponents, zeros up to 640 bytes;
* ``quant="latent"``: 512 codes, the 64 rotary values in 16 bits, 16 scale exponents, zeros up to 768 bytes.

A scale exponent e is held as the byte e + 127.
"""
import math

import torch

own = False

LATENT, ROPE, GROUP = 512, 64, 32
DIM = LATENT + ROPE
SCALE = 192 ** -0.5   # heads of 128 + 64 before the latent projection is folded into the queries
ROW_BYTES = {"none": 1152, "latent": 768, "row": 640}
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def attend(reqs, draft, heads, top_k, slots, dtype, quant, holes=0.0, tree=True, empty=False, name=None):
    """``slots``: of each request's part of the hot buffer; ``holes``: share of the selection that holds no position;
    ``tree``: the drafted tokens' own rows are read; ``empty``: the first request has selected nothing, and the first
    drafted token of each does not see itself either."""
    c = dict(kind="attend", reqs=reqs, draft=draft, heads=heads, top_k=top_k, slots=slots, dtype=dtype, quant=quant,
             holes=holes, tree=tree, empty=empty)
    if name is not None:
        c["name"] = name
    return c


def rows(kind, reqs, per_req, slots, dtype, quant, holes=0.0, name=None):
    """``slots`` 0: the rows one after another, without slots."""
    c = dict(kind=kind, reqs=reqs, per_req=per_req, slots=slots, dtype=dtype, quant=quant, holes=holes)
    if name is not None:
        c["name"] = name
    return c


def listed():
    return [
        # the decode driver's default run (8 requests, 64 selected), one GPU's 16 heads: latency
        attend(8, 1, 16, 64, 64, "fp16", "none", tree=False, name="decode_default"),
        # sparse-attention decode of a full batch, every head, 16-bit rows
        attend(64, 1, 128, 2048, 4096, "bf16", "none", tree=False, name="decode_dsa"),
        # ... and 8-bit rows
        attend(64, 1, 128, 2048, 4096, "bf16", "row", tree=False, name="decode_dsa_8bit"),
        # ... with the heads spread over eight GPUs, rotary part in 16 bits
        attend(64, 1, 16, 2048, 4096, "bf16", "latent", tree=False, name="decode_dsa_16_heads"),
        # one request alone: few queries, the selection has to be spread over the GPU
        attend(1, 2, 128, 2048, 4096, "bf16", "none", name="decode_one_request"),
        # drafted trees of eight tokens, every head: the matrix products bound it
        attend(16, 8, 128, 2048, 4096, "fp16", "row", name="tree_dsa_8bit"),
        # the largest selection (the slot limit's), large trees
        attend(4, 32, 128, 8192, 65518, "bf16", "none", name="tree_slot_limit"),
        # odd sizes, holes in the selection, drafted tokens that see nothing
        attend(5, 7, 20, 333, 1000, "fp16", "latent", holes=0.3, empty=True, name="tree_ragged"),
        # the new token's row of each request, to its slot
        rows("write", 64, 1, 4104, "bf16", "row", name="write_decode"),
        # one prompt's rows in every layer (61 x 8192), before their export
        rows("write", 1, 61 * 8192, 0, "fp16", "latent", name="write_prompt"),
        # a small selection read back, with holes
        rows("read", 8, 64, 64, "bf16", "latent", holes=0.1, name="read_default"),
        # a full batch's selection read back
        rows("read", 64, 2048, 4096, "bf16", "row", name="read_dsa"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype, quant = rng.choice(["bf16", "fp16"]), rng.choice(["none", "latent", "row"])
    kind = rng.choice(["attend", "attend", "attend", "write", "read"])
    if kind != "attend":
        quant = quant if quant != "none" else "row"
        n, reqs = _log_int(rng, 1, 400000), _log_int(rng, 1, 64)
        if rng.random() < 0.3:
            return rows(kind, 1, n, 0, dtype, quant)
        per = max(1, min(n // reqs, 4096))
        return rows(kind, reqs, per, per + rng.randrange(per + 64), dtype, quant, holes=rng.choice([0.0, 0.1]))
    reqs, heads, top_k = _log_int(rng, 1, 64), rng.choice([1, 8, 16, 20, 32, 64, 96, 128]), _log_int(rng, 1, 8192)
    draft = rng.choice([1, 1, 1, 2, 4, _log_int(rng, 1, 64)])
    # at most half of the largest listed case's products
    while reqs * draft * heads * top_k > 1 << 26:
        draft, reqs = (draft + 1) // 2 if draft > 1 else 1, reqs if draft > 1 else (reqs + 1) // 2
    tree = draft > 1 or rng.random() < 0.3
    return attend(reqs, draft, heads, top_k, min(65518, top_k + rng.randrange(top_k + 64)), dtype, quant,
                  holes=rng.choice([0.0, 0.0, 0.05, 0.5]), tree=tree, empty=tree and rng.random() < 0.2)


# ---- what a user's program has in hand ----

def _pad16(n):
    return -(-n // 16) * 16


def _stride(c):
    """Rows of one request's part of the hot buffer: its slots, and the places of its drafted tokens behind them."""
    return _pad16(c["slots"]) + (c["draft"] if c["kind"] == "attend" and c["tree"] else 0)


def _values(n, dtype, gen):
    """Latent rows: a few channels larger than the others, rows of different magnitude."""
    x = torch.randn((n, DIM), generator=gen, device="cuda", dtype=torch.float32)
    x *= torch.exp(0.5 * torch.randn((1, DIM), generator=gen, device="cuda"))
    x *= torch.exp(0.3 * torch.randn((n, 1), generator=gen, device="cuda"))
    return x.to(dtype)


def _choose(reqs, count, slots, holes, gen):
    """int32 [reqs, count]: distinct slots in random order, a share of them -1."""
    at = torch.rand((reqs, slots), generator=gen, device="cuda").argsort(dim=1)[:, :count].to(torch.int32)
    if holes:
        at = at.masked_fill(torch.rand((reqs, count), generator=gen, device="cuda") < holes, -1)
    return at.contiguous()


def _tree(reqs, draft, gen):
    """int64 [reqs, draft]: bit j of token i says that i sees j: its ancestors and itself; a token's parent is one of
    the four before it."""
    up = torch.randint(1, 5, (reqs, draft), generator=gen, device="cuda")
    mask = torch.zeros((reqs, draft), dtype=torch.int64, device="cuda")
    mask[:, 0] = 1
    for i in range(1, draft):
        parent = (i - up[:, i:i + 1]).clamp(min=0)
        mask[:, i] = mask.gather(1, parent)[:, 0] | (-(1 << 63) if i == 63 else 1 << i)
    return mask


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    dtype, quant, reqs = DTYPES[c["dtype"]], c["quant"], c["reqs"]
    s = {"case": c, "stride": _stride(c)}
    if c["kind"] == "attend":
        B, T, H = reqs, c["draft"], c["heads"]
        s["hot"] = _encode(_values(B * s["stride"], dtype, gen), quant)
        s["q"] = torch.randn((B, T, H, DIM), generator=gen, device="cuda").to(dtype)
        s["slots"] = _choose(B, c["top_k"], c["slots"], c["holes"], gen)
        s["draft_slots"] = s["tree_mask"] = None
        if c["tree"]:
            places = _pad16(c["slots"]) + torch.arange(T, dtype=torch.int32, device="cuda")
            s["draft_slots"], s["tree_mask"] = places.repeat(B, 1), _tree(B, T, gen)
        if c["empty"]:
            s["slots"][0] = -1
            s["tree_mask"][:, 0] = 0
        s["out"] = torch.empty((B, T, H, LATENT), dtype=dtype, device="cuda")
        s["lse"] = torch.empty((B, T, H), dtype=torch.float32, device="cuda")
        return s
    n = reqs * c["per_req"]
    s["slots"] = _choose(reqs, c["per_req"], c["slots"], c["holes"], gen) if c["slots"] else None
    total = reqs * s["stride"] if c["slots"] else n
    if c["kind"] == "write":
        s["rows"] = _values(n, dtype, gen)
        # what the buffer held before
        s["hot"] = _encode(_values(1, dtype, gen), quant).repeat(total, 1)
    else:
        s["hot"] = _encode(_values(total, dtype, gen), quant)
        s["out"] = torch.empty((n, DIM), dtype=dtype, device="cuda")
    return s


# ---- one pass ----

_xds = None


def _package():
    global _xds
    if _xds is None:
        from kv_offload_proto_amd import _kvops, xds

        try:
            _kvops.init(0, "")
        except RuntimeError as exc:
            if "already inited" not in str(exc):
                raise
        _xds = xds
    return _xds


def run(state):
    s, c = state, state["case"]
    if own:
        xds = _package()
        fmt = xds.row_format(DTYPES[c["dtype"]], LATENT, ROPE, c["quant"])
        if c["kind"] == "attend":
            xds.tree_attention(fmt, s["q"], s["hot"], s["slots"], SCALE, req_stride_rows=s["stride"],
                               draft_slots=s["draft_slots"], tree_mask=s["tree_mask"], out=s["out"], lse=s["lse"])
            return {"out": s["out"], "lse": s["lse"]}
        if c["kind"] == "write":
            xds.quantize_rows(fmt, s["rows"], s["hot"], s["slots"], req_stride_rows=s["stride"])
            return _parts(s["hot"], c["quant"], DTYPES[c["dtype"]])
        xds.dequantize_rows(fmt, s["hot"], s["slots"], req_stride_rows=s["stride"], out=s["out"])
        return s["out"]
    if c["kind"] == "attend":
        return _attend(s, c)
    if c["kind"] == "write":
        rec, n = _encode(s["rows"], c["quant"]), s["rows"].shape[0]
        if s["slots"] is None:
            s["hot"][:n] = rec
        else:
            at = _row_of(s["slots"], s["stride"]).reshape(-1)
            s["hot"][at[at >= 0]] = rec[at >= 0]
        return _parts(s["hot"], c["quant"], DTYPES[c["dtype"]])
    if s["slots"] is None:
        return _decode(s["hot"], c["quant"], DTYPES[c["dtype"]]).to(DTYPES[c["dtype"]])
    at = _row_of(s["slots"], s["stride"]).reshape(-1)
    x = _decode(s["hot"][at.clamp(min=0)], c["quant"], DTYPES[c["dtype"]])
    return torch.where((at >= 0)[:, None], x, 0.0).to(DTYPES[c["dtype"]])


# ---- the plain forms ----

def _row_of(slots, stride):
    """Hot row of each slot (request b's slot s is row b * stride + s), -1 where there is none."""
    base = torch.arange(slots.shape[0], device=slots.device)[:, None] * stride
    return torch.where(slots >= 0, slots.to(torch.int64) + base, -1)


def _encode(x, quant):
    """uint8 [n, row bytes] of 16-bit rows [n, 576]."""
    raw = x.contiguous().view(torch.uint8)
    if quant == "none":
        return raw
    n, d = x.shape[0], LATENT if quant == "latent" else DIM
    rec = torch.zeros((n, ROW_BYTES[quant]), dtype=torch.uint8, device=x.device)
    g = x[:, :d].to(torch.float32).reshape(n, d // GROUP, GROUP)
    mant, exp = torch.frexp(torch.where(torch.isfinite(g), g.abs(), 0.0).amax(dim=2))
    e = torch.where(mant > 0, exp - 9 + (mant > 0.875), -127).clamp(-127, 127)
    codes = torch.ldexp(g, -e[:, :, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    rec[:, :d] = codes.reshape(n, d).view(torch.uint8)
    end = d + (DIM - d) * 2
    rec[:, d:end] = raw[:, 2 * d:]
    rec[:, end:end + d // GROUP] = (e + 127).to(torch.uint8)
    return rec


def _parts(rec, quant, dtype):
    """The values that the bytes of rows stand for: codes, scales, rotary part."""
    d = LATENT if quant == "latent" else DIM
    end = d + (DIM - d) * 2
    parts = {"codes": rec[:, :d].view(torch.float8_e4m3fn), "scales": rec[:, end:end + d // GROUP].view(torch.float8_e8m0fnu)}
    if d < DIM:
        parts["rope"] = rec[:, d:end].view(dtype)
    return parts


def _decode(rec, quant, dtype):
    """float32 [n, 576] of rows."""
    if quant == "none":
        return rec.view(dtype).to(torch.float32)
    d = LATENT if quant == "latent" else DIM
    end = d + (DIM - d) * 2
    codes = rec[:, :d].view(torch.float8_e4m3fn).to(torch.float32).reshape(-1, d // GROUP, GROUP)
    e = rec[:, end:end + d // GROUP].to(torch.int32) - 127
    x = torch.ldexp(codes, e[:, :, None]).reshape(-1, d)
    return torch.cat([x, rec[:, d:end].contiguous().view(dtype).to(torch.float32)], dim=1) if d < DIM else x


def _keys(s, c):
    """Hot rows [reqs, keys] that the queries read (-1: none), and bool [reqs, draft, keys]: which token sees which."""
    at = _row_of(s["slots"], s["stride"])
    seen = (at >= 0)[:, None, :].expand(-1, c["draft"], -1)
    if s["draft_slots"] is not None:
        bits = torch.arange(c["draft"], device=at.device)
        sees = ((s["tree_mask"][:, :, None] >> bits) & 1).bool()
        more = _row_of(s["draft_slots"], s["stride"])
        at, seen = torch.cat([at, more], dim=1), torch.cat([seen, sees & (more >= 0)[:, None, :]], dim=2)
    return at, seen


def _attend(s, c):
    B, T, H, dtype = c["reqs"], c["draft"], c["heads"], DTYPES[c["dtype"]]
    at, seen = _keys(s, c)
    k = _decode(s["hot"][at.clamp(min=0).reshape(-1)], c["quant"], dtype).reshape(B, -1, DIM)
    k = torch.where((at >= 0)[:, :, None], k, 0.0)
    q = s["q"].to(torch.float32).reshape(B, T * H, DIM)
    score = torch.bmm(q, k.transpose(1, 2).contiguous()).mul_(SCALE).reshape(B, T, H, -1)
    score.masked_fill_(~seen[:, :, None, :], -math.inf)
    top = score.amax(dim=3, keepdim=True)
    p = torch.exp(score.sub_(torch.where(top > -math.inf, top, 0.0)))
    total = p.sum(dim=3, keepdim=True)
    out = torch.bmm(p.reshape(B, T * H, -1), k[:, :, :LATENT].contiguous()).reshape(B, T, H, LATENT)
    out = out / torch.where(total > 0, total, 1.0)
    return {"out": out.to(dtype), "lse": (top + torch.log(total))[..., 0]}


# ---- the definitions in 64 bits ----

def _e4m3_exact(x):
    """Nearest value of the 8-bit code's grid (4 significant bits, steps of 2^-9 below 2^-6), ties to even."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))).clamp(max=8) - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def _parts_exact(x, quant):
    d = LATENT if quant == "latent" else DIM
    x = x.double()
    g = x[:, :d].reshape(x.shape[0], d // GROUP, GROUP)
    top = g.abs().amax(dim=2)
    scale = torch.exp2(torch.ceil(torch.log2(top.clamp(min=2.0 ** -140) / 448)).clamp(-127, 127))
    parts = {"codes": _e4m3_exact(g / scale[:, :, None]).reshape(-1, d), "scales": scale}
    if d < DIM:
        parts["rope"] = x[:, d:]
    return parts


def _values_exact(s, c, at):
    """float64 [n, 576] of the rows `at` of the hot buffer, from its bytes."""
    quant, dtype = c["quant"], DTYPES[c["dtype"]]
    rec = s["hot"][at]
    if quant == "none":
        return rec.view(dtype).double()
    d = LATENT if quant == "latent" else DIM
    end = d + (DIM - d) * 2
    b = torch.arange(256, device=rec.device)
    expo, frac = (b >> 3) & 15, (b & 7).double()
    table = torch.where(expo > 0, (8 + frac) * torch.exp2((expo - 10).double()), frac * 2.0 ** -9)
    table = torch.where(b >= 128, -table, table)
    x = table[rec[:, :d].long()].reshape(-1, d // GROUP, GROUP)
    x = (x * torch.exp2(rec[:, end:end + d // GROUP].double() - 127)[:, :, None]).reshape(-1, d)
    return torch.cat([x, rec[:, d:end].contiguous().view(dtype).double()], dim=1) if d < DIM else x


def exact(case, seed):
    s, c = prepare(case, seed), case
    at = None if s["slots"] is None else _row_of(s["slots"], s["stride"])
    if c["kind"] == "write":
        if at is None:
            return _parts_exact(s["rows"], c["quant"])
        held = _parts(s["hot"], c["quant"], DTYPES[c["dtype"]])
        new, at = _parts_exact(s["rows"], c["quant"]), at.reshape(-1)
        for name, part in new.items():
            whole = held[name].contiguous().double()
            whole[at[at >= 0]] = part[at >= 0]
            new[name] = whole
        return new
    if c["kind"] == "read":
        if at is None:
            return _values_exact(s, c, slice(None))
        at = at.reshape(-1)
        return torch.where((at >= 0)[:, None], _values_exact(s, c, at.clamp(min=0)), 0.0)
    at, seen = _keys(s, c)
    out, lse = [], []
    for b in range(c["reqs"]):
        k = _values_exact(s, c, at[b].clamp(min=0))
        score = torch.einsum("thd,nd->thn", s["q"][b].double(), k) * SCALE
        score = torch.where(seen[b][:, None, :], score, -math.inf)
        lse.append(torch.logsumexp(score, dim=2))
        p = torch.where(seen[b][:, None, :], torch.exp(score - lse[-1][..., None]), 0.0)
        out.append(torch.einsum("thn,nd->thd", p, k[:, :LATENT]))
    return {"out": torch.stack(out), "lse": torch.stack(lse)}


def work(case):
    c, row = case, ROW_BYTES[case["quant"]]
    if c["kind"] != "attend":
        n = round(c["reqs"] * c["per_req"] * (1 - c["holes"]))
        return {"bytes": n * row + c["reqs"] * c["per_req"] * (2 * DIM + (4 if c["slots"] else 0)), "flops": 0}
    queries = c["reqs"] * c["draft"] * c["heads"]
    keys = c["top_k"] * (1 - c["holes"])
    drafted = c["draft"] if c["tree"] else 0
    bytes_ = c["reqs"] * ((keys + drafted) * row + 4 * c["top_k"] + 12 * drafted) + queries * (2 * DIM + 2 * LATENT + 4)
    return {"bytes": round(bytes_), "flops": round(2 * queries * (keys + (1 if drafted else 0)) * (DIM + LATENT))}
