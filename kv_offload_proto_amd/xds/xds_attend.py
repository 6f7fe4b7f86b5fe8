"""Decode steps that attend: the data plane of ``xds_decode`` with rows in 8 bits
(or 16) and the attention over what it brought.

    python -m kv_offload_proto_amd.xds.xds_attend --quant row --steps 10

Each request holds a prompt in the host pool, as rows of the chosen form, and
drafts a random tree of tokens per step.  A step does, for every layer,

    quantize_rows    the drafted tokens' rows, into the slots of their positions
    sieve_update     slots of the selected positions (a stand-in for the indexer)
    batch_read_fused the missing rows, from the host segments
    tree_attention   every drafted token over the selection and its ancestors

then accepts one path of each tree: its rows move up to the positions that
follow the sequence, where later steps select them like any others.  Positions
past the prompt live behind the device buffer (slot padded + position - prompt
length, as ``sieve_update`` names them), so hot rows are strided by the padded
buffer and room for every token that the run can add.

Unless ``--no-check`` is given each output is compared with the formula in 64
bits on the rows that were exported, addressed by the position that owns each
slot: a missing import, a row that moved wrongly or a mistake of a kernel all
show.  A SIEVE sweep that laps the buffer can take a slot that it handed out
earlier in the same update; the later position then owns it, and the step's
line counts such positions as displaced.
The reference's driver ends at the import (xds/xds_decode.py:224-270).
"""
import argparse
import sys
import time

import numpy as np


def parse_args(argv=None):
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    p.add_argument("--device", type=int, default=0)
    p.add_argument("--quant", choices=("none", "latent", "row"), default="row")
    p.add_argument("--dtype", choices=("bf16", "fp16"), default="bf16")
    p.add_argument("--layers", type=int, default=2)
    p.add_argument("--req-num", type=int, default=8)
    p.add_argument("--prefill", type=int, default=256)
    p.add_argument("--topk", type=int, default=64)
    p.add_argument("--device-buffer-size", type=int, default=128, help="slots; fewer than twice topK are often taken "
                   "again within one update")
    p.add_argument("--heads", type=int, default=16)
    p.add_argument("--draft", type=int, default=4, help="tokens drafted per step (1: plain decoding)")
    p.add_argument("--node-num", type=int, default=2)
    p.add_argument("--steps", type=int, default=10)
    p.add_argument("--seed", type=int, default=42)
    p.add_argument("--no-check", action="store_true")
    args = p.parse_args(argv)
    if not 1 <= args.draft <= 64:
        p.error("--draft must be in [1, 64]")
    return args


def draw_tree(rng, reqs, tokens):
    """Parents (-1: the sequence's last token) and bit masks of each token's ancestors and itself."""
    parent = np.full((reqs, tokens), -1, np.int64)
    mask = np.zeros((reqs, tokens), np.uint64)
    for b in range(reqs):
        for t in range(tokens):
            parent[b, t] = rng.integers(max(-1, t - 3), t)
            up = mask[b, parent[b, t]] if parent[b, t] >= 0 else np.uint64(0)
            mask[b, t] = up | np.uint64(1 << t)
    return parent, mask.view(np.int64)


def draw_selection(rng, prefill, seq_lens, top_k):
    """Distinct positions of every sequence, its newest among them, padded with -1."""
    out = np.full((len(seq_lens), top_k), -1, np.int32)
    for b, n in enumerate(seq_lens):
        new = np.arange(max(prefill, n - top_k // 2), n)
        old = rng.permutation(prefill)[:top_k - len(new)]
        out[b, :len(new) + len(old)] = rng.permutation(np.concatenate([new, old]))
    return out


def expected(q, keys, sees, scale):
    """float64 (out, lse, sum p |v|, largest sum |q k|) of one request: q [tokens, heads, dim], keys [n, dim],
    sees bool [tokens, n]."""
    import torch

    s = torch.matmul(q, keys.t()) * scale
    s = s.masked_fill(~sees[:, None, :], float("-inf"))
    lse = torch.logsumexp(s, dim=-1)
    p = torch.exp(s - lse[..., None])
    v = keys[:, :512].contiguous()
    size = (torch.matmul(q.abs(), keys.abs().t()) * scale).amax(dim=-1)
    return torch.matmul(p, v), lse, torch.matmul(p, v.abs()), size


def main(argv=None):
    args = parse_args(argv)
    import torch

    if not torch.cuda.is_available():
        print("[xds][ERROR] no GPU visible")
        return 1
    from ..kvops_ext import _kvops
    from .xds_attention import dequantize_rows, quantize_rows, row_format, tree_attention
    from .xds_offload import XdsOffloadCoordinator
    from .xds_seg_pool import HostSegPool

    rng = np.random.default_rng(args.seed)
    dtype = torch.bfloat16 if args.dtype == "bf16" else torch.float16
    unit = 2.0 ** (-8 if args.dtype == "bf16" else -11)          # half a step of the type
    fmt = row_format(dtype, quant=args.quant)
    L, R, T, H, prefill, top_k = args.layers, args.req_num, args.draft, args.heads, args.prefill, args.topk
    dev = torch.device("cuda", args.device)
    torch.cuda.set_device(dev)
    stream = torch.cuda.current_stream().cuda_stream
    scale = fmt.dim ** -0.5

    gen = torch.Generator(device=dev)
    gen.manual_seed(args.seed)

    def store(rows, hot, slots=None, stride=0):
        """16-bit rows into hot rows of the form."""
        if args.quant != "none":
            quantize_rows(fmt, rows, hot, slots, stride, stream=stream)
        elif slots is None:
            hot.view(dtype)[:rows.shape[0]] = rows
        else:
            first = torch.arange(slots.shape[0], device=dev)[:, None] * stride
            hot.view(dtype)[(slots + first).reshape(-1)] = rows

    def values(hot):
        return hot.view(dtype) if args.quant == "none" else dequantize_rows(fmt, hot, dtype=torch.float32)

    pool = HostSegPool(args.device, L, R * prefill, fmt.row_bytes, node_num=args.node_num)
    pool.create_pool()
    try:
        # prompts: rows in their form, to the host segments
        src = torch.zeros((L, R * prefill, fmt.row_bytes), dtype=torch.uint8, device=dev)
        for l in range(L):
            store(torch.randn((R * prefill, fmt.dim), generator=gen, device=dev).to(dtype), src[l])
        pool.wait(pool.batch_write_alllayers(0, R * prefill, src, R * prefill * fmt.row_bytes, stream=stream))
        # the rows of every position, by layer and request, for the check
        known = None if args.no_check else [
            [list(x) for x in values(src[l]).double().cpu().reshape(R, prefill, fmt.dim)] for l in range(L)]
        del src
        coord = XdsOffloadCoordinator(dev, L, R, args.device_buffer_size, top_k, R, prefill)
        tail = coord.padded_buffer_size
        stride = tail + (args.steps + 1) * T
        for r in range(R):
            coord.admit_request(r, r, prefill, r * prefill, stream=stream)
        hot = torch.zeros((L, R * stride, fmt.row_bytes), dtype=torch.uint8, device=dev)
        # slot s of an admitted request holds token s: bring those rows, as a first selection of them all would
        first = min(prefill, args.device_buffer_size)
        resident = torch.arange(first, dtype=torch.int32, device=dev).expand(R, first).contiguous()
        ones = torch.ones((R, first), dtype=torch.int8, device=dev)
        req_pool = torch.arange(R, dtype=torch.int64, device=dev)
        seq_lens = np.full(R, prefill, np.int64)
        coord.set_batch(req_pool, torch.full((R,), prefill, dtype=torch.int32, device=dev))
        for l in range(L):
            pool.wait(pool.batch_read_fused(l, resident, req_pool, coord.req_host_base, resident, ones, coord.num_real,
                                            hot[l], R, first, stream=stream, hot_req_stride_rows=stride))
        print("[xds] {} requests of {} positions, {} layers, {!r}".format(R, prefill, L, fmt), flush=True)

        total_miss, worst = 0, 0.0
        for step in range(args.steps):
            parent, mask = draw_tree(rng, R, T)
            topk = draw_selection(rng, prefill, seq_lens, top_k)
            draft = (tail + seq_lens[:, None] - prefill + np.arange(T)).astype(np.int32)
            topk_d, draft_d, mask_d = (torch.from_numpy(x).to(dev) for x in (topk, draft, mask))
            coord.set_batch(req_pool, torch.from_numpy(seq_lens.astype(np.int32)).to(dev))
            rows = torch.randn((L, R * T, fmt.dim), generator=gen, device=dev).to(dtype)
            q = torch.randn((L, R, T, H, fmt.dim), generator=gen, device=dev).to(dtype)
            torch.cuda.synchronize()
            t0, miss, got, slots = time.perf_counter(), [], [], []
            for l in range(L):
                store(rows[l], hot[l], draft_d, stride)
                coord.sieve_update(l, topk_d, stream=stream)
                st = pool.batch_read_fused(l, topk_d, req_pool, coord.req_host_base, coord.top_k_device_slots,
                                           coord.is_miss, coord.num_real, hot[l], R, top_k, stream=stream,
                                           hot_req_stride_rows=stride)
                got.append(tree_attention(fmt, q[l], hot[l], coord.top_k_device_slots, scale, stride,
                                          draft_slots=draft_d, tree_mask=mask_d))
                slots.append(coord.top_k_device_slots.clone())
                miss.append(coord.miss_count())
                pool.wait(st)
            torch.cuda.synchronize()
            dt = time.perf_counter() - t0
            n_miss, displaced = int(sum(m.item() for m in miss)), 0
            total_miss += n_miss

            if not args.no_check:
                tree = (mask[:, :, None] >> np.arange(T)) & 1
                for l in range(L):
                    new = values(hot[l])[(draft_d + torch.arange(R, device=dev)[:, None] * stride).long()].double().cpu()
                    owner, at = coord.device_buffer_tokens[l].cpu().numpy(), slots[l].cpu().numpy()
                    for r in range(R):
                        pos = np.where(at[r] < tail, owner[r][np.clip(at[r], 0, tail - 1)], prefill + at[r] - tail)
                        pos = np.where(at[r] < 0, -1, pos)
                        displaced += int((pos != topk[r]).sum())
                        use = [known[l][r][p] for p in pos if p >= 0]
                        keys = torch.cat([torch.stack(use), new[r]])
                        sees = torch.cat([torch.ones((T, len(use)), dtype=torch.bool), torch.from_numpy(tree[r] != 0)], 1)
                        want, want_lse, size, score = expected(q[l, r].double().cpu(), keys, sees, scale)
                        # rounded weights and output, weights under fp16's range; a score's 576 products in 32 bits
                        off = fmt.dim * 2.0 ** -23 * score
                        lost = len(keys) * 2.0 ** -25 * keys[:, :512].abs().max() if args.dtype == "fp16" else 0.0
                        tol = unit * want.abs() + (unit + 2 * off + 2.0 ** -18)[..., None] * size + lost
                        err = ((got[l][0][r].double().cpu() - want).abs() / tol).max().item()
                        err_lse = ((got[l][1][r].double().cpu() - want_lse).abs() /
                                   (off + 2.0 ** -20 * (1 + want_lse.abs()))).max().item()
                        worst = max(worst, err, err_lse)
                        if not max(err, err_lse) <= 1.01:
                            print("[xds][ERROR] attention of step {} layer {} request {} is off: {:.2f} and {:.2f} of the "
                                  "rounding's bound".format(step, l, r, err, err_lse))
                            return 1
                        known[l][r].extend(new[r, i] for i in _path(parent[r], T - 1))

            # accept the path to each tree's last token: its rows move up behind the sequence
            src_rows, dst_rows = [], []
            for r in range(R):
                path = _path(parent[r], T - 1)
                at = r * stride + tail + int(seq_lens[r]) - prefill
                src_rows += [at + i for i in path]
                dst_rows += range(at, at + len(path))
                seq_lens[r] += len(path)
            src_d, dst_d = (torch.tensor(x, dtype=torch.int64, device=dev) for x in (src_rows, dst_rows))
            hot[:, dst_d] = hot[:, src_d]
            print("[xds] step {}: miss={} rows of {} bytes, {} tokens accepted, {:.1f} us a layer{}".format(
                step, n_miss, fmt.row_bytes, len(src_rows), dt * 1e6 / L,
                ", {} positions displaced".format(displaced) if displaced else ""), flush=True)
        if _kvops.read_overflow() != 0:
            print("[xds][ERROR] tail slot {:#x}".format(_kvops.read_overflow()))
            return 1
        print("[xds] summary: {} miss rows, {} B over the host link ({} B in 16 bits){}".format(
            total_miss, total_miss * fmt.row_bytes, total_miss * 2 * fmt.dim,
            "" if args.no_check else ", largest error {:.2f} of the rounding's bound".format(worst)))
    finally:
        pool.destroy()
    print("[xds] all done")
    return 0


def _path(parent, t):
    """Tokens from the root to t, in order."""
    path = []
    while t >= 0:
        path.append(int(t))
        t = parent[t]
    return path[::-1]


if __name__ == "__main__":
    sys.exit(main())
