"""tree_attention at sizes where a workgroup takes 64 or 128 queries, against the formula in 64 bits."""
import numpy as np
import pytest
import torch

import row_model as rm
from test_gpu_attention import SCALE, check, dev, problem, raw_values, run

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _lib(kvops):
    yield
    torch.cuda.synchronize()


def model(p, scale=SCALE):
    """As row_model.attention, with the products in 64 bits on the GPU."""
    hot = rm.decode(p["hot"].numpy(), raw_values(p["dtype"]), p["quant"])
    B, T, H, _ = p["q"].shape
    out, lse = np.zeros((B, T, H, rm.LATENT)), np.full((B, T, H), -np.inf)
    weighted, size = np.zeros((B, T, H, rm.LATENT)), np.zeros((B, T, H))
    for b, (rows, seen) in enumerate(rm.keys_of(p["slots"], p["draft_slots"], p["tree_mask"], p["stride"], len(hot))):
        if not len(rows):
            continue
        k = torch.from_numpy(hot[rows]).cuda()
        q = p["q"][b].double().cuda().reshape(T * H, -1)
        sees = torch.from_numpy(np.broadcast_to(seen, (T, len(rows)))).cuda().repeat_interleave(H, 0)
        s = torch.mm(q, k.t()) * scale
        s = torch.where(sees, s, float("-inf"))
        some = sees.any(1, keepdim=True)
        total = torch.logsumexp(s, 1, keepdim=True)
        w = torch.where(some, torch.exp(s - total), 0.0)
        v = k[:, :rm.LATENT].contiguous()
        each = torch.where(sees, torch.mm(q.abs(), k.abs().t()) * abs(scale), 0.0)
        out[b] = torch.mm(w, v).cpu().numpy().reshape(out[b].shape)
        weighted[b] = torch.mm(w, v.abs()).cpu().numpy().reshape(out[b].shape)
        lse[b] = total.cpu().numpy().reshape(T, H)
        size[b] = each.amax(1).cpu().numpy().reshape(T, H)
    return out, lse, weighted, size


CASES = [
    # requests, tokens, heads, topK, slots, dtype, quant, tree, holes
    (70, 1, 128, 301, 320, "bf16", "none", False, 0.02),
    (70, 1, 127, 64, 100, "fp16", "row", False, 0),
    (70, 1, 128, 33, 48, "bf16", "latent", True, 0.3),
    (33, 2, 128, 2, 5, "bf16", "latent", True, 0.3),
    (40, 3, 100, 333, 400, "fp16", "none", True, 0.1),
    (64, 1, 128, 700, 720, "fp16", "none", False, 0),
    (5, 64, 64, 300, 310, "bf16", "row", True, 0.05),
    (6, 33, 127, 65, 80, "bf16", "none", True, 0.2),
    (5, 50, 60, 2200, 2300, "bf16", "none", True, 0),
    (5, 64, 64, 2500, 2600, "fp16", "none", True, 0),
    (3, 64, 128, 150, 160, "fp16", "latent", True, 0),
    (4, 32, 128, 1500, 1600, "bf16", "none", True, 0.01),
    (16, 8, 127, 1200, 1300, "fp16", "none", True, 0),
    (8, 16, 128, 1400, 1410, "bf16", "row", False, 0),
    (32, 1, 128, 1100, 1200, "fp16", "none", False, 0.05),
    (4, 32, 128, 4200, 4300, "bf16", "none", True, 0),
]


@pytest.mark.parametrize("reqs,tokens,heads,top_k,slots,dtype,quant,tree,holes", CASES)
def test_many_queries(reqs, tokens, heads, top_k, slots, dtype, quant, tree, holes):
    p = problem(reqs, tokens, heads, top_k, slots, dtype, quant, tree, holes)
    out, lse = run(p)
    check(p, out, lse, expected=model(p))
    again, lse2 = run(p)
    assert torch.equal(out, again) and torch.equal(lse, lse2)


@pytest.mark.parametrize("reqs,tokens,heads", [(70, 1, 128), (5, 64, 64)])
@pytest.mark.parametrize("dtype,quant", [("bf16", "none"), ("fp16", "row")])
def test_scores_far_apart(reqs, tokens, heads, dtype, quant):
    p = problem(reqs, tokens, heads, 200, 210, dtype, quant, tokens > 1, q_scale=30.0)
    check(p, *run(p), expected=model(p))


@pytest.mark.parametrize("reqs,tokens,heads", [(70, 2, 128), (5, 64, 64)])
@pytest.mark.parametrize("dtype,quant", [("bf16", "none"), ("fp16", "latent"), ("bf16", "row")])
def test_unseen_rows_have_no_effect(reqs, tokens, heads, dtype, quant):
    """NaN in every row that no query sees, in the row that one token alone sees, and a token that sees nothing."""
    p = problem(reqs, tokens, heads, 90, 100, dtype, quant, True, holes=0.2)
    p["slots"][1] = -1
    p["tree_mask"][1, 1] = 0
    p["tree_mask"][2, :] &= np.uint64(2 ** 64 - 2)           # token 0's row of request 2: no one's
    p["draft_slots"][3, 1] = -1
    clean = run(p)
    check(p, *clean, expected=model(p))
    used = set()
    for rows, seen in rm.keys_of(p["slots"], p["draft_slots"], p["tree_mask"], p["stride"], p["hot"].shape[0]):
        used |= {int(r) for r, s in zip(rows, seen.T) if s.any()}
    hot = p["hot"].clone()
    hot[[r for r in range(hot.shape[0]) if r not in used]] = 0xFF
    for got, want in zip(run(p, hot=hot), clean):
        assert torch.equal(got, want)
    # token 0's row of request 4 is a NaN: whoever sees it has one, the others what they had
    p["tree_mask"][4, 1] = np.uint64(2)
    clean = run(p)
    hot = p["hot"].clone()
    hot[4 * p["stride"] + int(p["draft_slots"][4, 0])] = 0xFF
    out, lse = run(p, hot=hot)
    sees = (p["tree_mask"] & np.uint64(1)) != 0
    sees[:4] = sees[5:] = False
    sees = torch.from_numpy(sees).cuda()
    assert bool(torch.isnan(out[sees]).any()) and bool(torch.isnan(lse[sees]).all())
    assert torch.equal(out[~sees], clean[0][~sees]) and torch.equal(lse[~sees], clean[1][~sees])
