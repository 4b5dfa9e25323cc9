"""What is measured of the serving operators: appending a batch of ragged chunks to a paged KV cache with the rotary
position rotation on the way, attention of those chunks over the cache, and drawing the next tokens from the logits.

A case names an operator and its sizes; the sequence lengths of a case follow from the case alone, the values from the
seed.  `run` computes the operator with elementary torch operations, or (`own`) with the framework's entry points."""
import math
import random

import numpy as np
import torch

own = False

_CACHE = dict(heads=32, kv_heads=8, head_dim=128, block=16)   # the attention shape of the 8B decoder that bench.py runs
_SMALL = dict(heads=12, kv_heads=12, head_dim=64, block=16)   # the 12-head, 768-wide decoder of the tests


def listed():
    return [
        # one decode step of the benchmark's batch: every sequence appends one token
        dict(name="append step", op="append", dtype="f32", seqs=128, chunked=0, chunk_lo=1, chunk_hi=1, step=1, prefix_lo=256, prefix_hi=2048, lens=1, rotary=128, pairs="half", **_CACHE),
        # prompts of the longest prefill pass, several at once
        dict(name="append prompts", op="append", dtype="f32", seqs=4, chunked=4, chunk_lo=2048, chunk_hi=2048, step=1, prefix_lo=0, prefix_hi=0, lens=2, rotary=128, pairs="half", **_CACHE),
        # ragged prompts of a small multi-head model: adjacent pairs, half of each head rotated, bf16 activations
        dict(name="append ragged bf16", op="append", dtype="bf16", seqs=19, chunked=19, chunk_lo=1, chunk_hi=1501, step=1, prefix_lo=0, prefix_hi=700, lens=3, rotary=32, pairs="adjacent", **_SMALL),
        # a few drafted tokens of eight sequences are checked at once
        dict(name="attention drafts bf16", op="attention", dtype="bf16", seqs=8, chunked=0, chunk_lo=1, chunk_hi=1, step=4, prefix_lo=200, prefix_hi=1000, lens=4, **_CACHE),
        # one decode step of the benchmark's batch
        dict(name="attention step", op="attention", dtype="f32", seqs=128, chunked=0, chunk_lo=1, chunk_hi=1, step=1, prefix_lo=256, prefix_hi=2048, lens=5, **_CACHE),
        # continuous batching: four prompts advance by a chunk while sixty sequences decode
        dict(name="attention mixed", op="attention", dtype="f32", seqs=64, chunked=4, chunk_lo=257, chunk_hi=512, step=1, prefix_lo=256, prefix_hi=2048, lens=6, **_CACHE),
        # fresh prompts, 16-bit activations
        dict(name="attention prompts bf16", op="attention", dtype="bf16", seqs=4, chunked=4, chunk_lo=2048, chunk_hi=2048, step=1, prefix_lo=0, prefix_hi=0, lens=7, **_CACHE),
        # one chunk of a long document, odd lengths
        dict(name="attention long bf16", op="attention", dtype="bf16", seqs=1, chunked=1, chunk_lo=2039, chunk_hi=2039, step=1, prefix_lo=30011, prefix_hi=30011, lens=8, **_CACHE),
        # prompts of the small multi-head model in 32 bits
        dict(name="attention small prompts", op="attention", dtype="f32", seqs=16, chunked=16, chunk_lo=300, chunk_hi=1024, step=1, prefix_lo=0, prefix_hi=64, lens=9, **_SMALL),
        # the next token of one sequence from the 8B decoder's vocabulary
        dict(name="sample one", op="sample", dtype="f32", rows=1, vocab=128256, stride=128256, k_lo=0, k_hi=0, p=0.9, min_p=0.0, masked=0.0),
        # the next tokens of the benchmark's batch, every filter in use
        dict(name="sample batch", op="sample", dtype="f32", rows=128, vocab=128256, stride=128256, k_lo=0, k_hi=1000, p=0.95, min_p=0.02, masked=0.0),
        # many rows of a small vocabulary in 16 bits (ties), half of it masked as by a grammar, rows further apart than they are long
        dict(name="sample masked bf16", op="sample", dtype="bf16", rows=512, vocab=32000, stride=32008, k_lo=1, k_hi=50, p=0.9, min_p=0.0, masked=0.5),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attention", "sample"])
    dtype = rng.choice(["f32", "bf16"])
    if op == "sample":
        vocab = _spread(rng, 1000, 128256)
        rows = _spread(rng, 1, max(1, min(512, 128 * 128256 // vocab)))
        k = rng.choice([0, 0, 1, _spread(rng, 2, 2000)])
        return dict(op=op, dtype=dtype, rows=rows, vocab=vocab, stride=vocab + rng.choice([0, 1, 7, 64]), k_lo=min(k, 1), k_hi=k,
                    p=rng.choice([1.0, round(rng.uniform(0.3, 0.999), 3)]), min_p=rng.choice([0.0, round(rng.uniform(0.001, 0.2), 4)]),
                    masked=rng.choice([0.0, 0.0, 0.9]))
    head_dim = rng.choice([64, 128])
    kv_heads = rng.choice([1, 2, 4, 8])
    shape = dict(heads=kv_heads * rng.choice([1, 2, 3, 4, 8]), kv_heads=kv_heads, head_dim=head_dim, block=rng.choice([16, 16, 32, 64]))
    seqs = _spread(rng, 1, 128)
    chunked = rng.choice([0, seqs, max(1, seqs // 8)])
    longest = _spread(rng, 2, max(2, 4096 // max(1, chunked)))
    # at most the work of the longest listed case, in the plain form's padded batch too
    most = 2_000_000_000 // (shape["heads"] * seqs * (longest if chunked else 5)) - longest
    prefix = _spread(rng, 1, max(1, min(most, 65536 // seqs if op == "attention" else 8192 // seqs)))
    case = dict(op=op, dtype=dtype, seqs=seqs, chunked=chunked, chunk_lo=max(1, longest // 3), chunk_hi=longest, step=rng.choice([1, 1, 2, 5]),
                prefix_lo=prefix // 4, prefix_hi=prefix, lens=rng.randrange(1 << 30), **shape)
    if op == "append":
        case.update(rotary=rng.choice([head_dim, head_dim // 2]), pairs=rng.choice(["half", "adjacent"]))
    return case


# ------------------------------------------------------------------------------------------------ sizes that follow from a case


def _lengths(case):
    """New tokens and cached tokens (the new ones among them) of every sequence; the first `chunked` sequences bring a chunk each."""
    r = random.Random(case["lens"])
    new = [r.randint(case["chunk_lo"], case["chunk_hi"]) if b < case["chunked"] else case["step"] for b in range(case["seqs"])]
    return new, [n + r.randint(case["prefix_lo"], case["prefix_hi"]) for n in new]


def _item(case):
    return 4 if case["dtype"] == "f32" else 2


def work(case):
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        # the logits once, five parameters in, three values out; a subtraction, an exponential and an addition per logit
        return dict(bytes=rows * vocab * _item(case) + rows * 4 * 8, flops=3.0 * rows * vocab)
    new, total = _lengths(case)
    rows, heads, kv, d = sum(new), case["heads"], case["kv_heads"], case["head_dim"]
    index = 4 * (2 * case["seqs"] + 1 + sum(-(-t // case["block"]) for t in total))
    if case["op"] == "append":
        moved = rows * ((2 * heads + 2 * kv) * d * _item(case) + 2 * kv * d * 2 + case["rotary"] * 4)
        return dict(bytes=moved + index, flops=3.0 * rows * (heads + kv) * case["rotary"])
    pairs = sum(n * (t - n) + n * (n + 1) // 2 for n, t in zip(new, total))
    return dict(bytes=2 * rows * heads * d * _item(case) + 2 * sum(total) * kv * d * 2 + index, flops=4.0 * d * heads * pairs)


# ------------------------------------------------------------------------------------------------ inputs


def _values(case, gen, *shape):
    x = torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)
    return x if case["dtype"] == "f32" else x.to(torch.bfloat16)


def _prepare_sample(case, gen):
    rows, vocab = case["rows"], case["vocab"]
    x = torch.randn(rows, case["stride"], generator=gen, device="cuda") * 2.5
    # a few likely continuations stand out of every row, as in a trained model's logits
    x.scatter_add_(1, torch.randint(0, vocab, (rows, 24), generator=gen, device="cuda"), 6.0 * torch.rand(rows, 24, generator=gen, device="cuda"))
    if case["masked"]:
        x.masked_fill_(torch.rand(rows, case["stride"], generator=gen, device="cuda") < case["masked"], -math.inf)
    st = dict(logits=x if case["dtype"] == "f32" else x.to(torch.bfloat16))
    st["temperature"] = 0.6 + 0.6 * torch.rand(rows, generator=gen, device="cuda")
    st["top_k"] = torch.randint(case["k_lo"], case["k_hi"] + 1, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    st["top_p"] = torch.full((rows,), case["p"], device="cuda")
    st["min_p"] = torch.full((rows,), case["min_p"], device="cuda")
    st["u"] = torch.rand(rows, generator=gen, device="cuda")
    st["ids"] = torch.zeros(rows, dtype=torch.int32, device="cuda")
    st["prob"] = torch.zeros(rows, device="cuda")
    st["kept"] = torch.zeros(rows, dtype=torch.int32, device="cuda")
    return st


def _prepare_cache(case, gen):
    new, total = _lengths(case)
    kv, d, block = case["kv_heads"], case["head_dim"], case["block"]
    used = [-(-t // block) for t in total]
    blocks = sum(used) + 3
    order = torch.randperm(blocks, generator=gen, device="cuda").to(torch.int32)
    tables = torch.full((case["seqs"], max(used)), -1, dtype=torch.int32, device="cuda")   # -1: a slot not in use
    at = torch.tensor([0] + used, device="cuda").cumsum(0)
    col = torch.arange(max(used), device="cuda")
    inside = col < torch.tensor(used, device="cuda")[:, None]
    tables[inside] = order[(at[:-1, None] + col)[inside]]
    st = dict(tables=tables, q_starts=torch.tensor([0] + new, device="cuda").cumsum(0).to(torch.int32),
              seq_lens=torch.tensor(total, dtype=torch.int32, device="cuda"))
    for name in ("k_pool", "v_pool"):
        st[name] = torch.randn(blocks, block, kv * d, generator=gen, device="cuda", dtype=torch.float32).to(torch.bfloat16)
    return st, sum(new), max(new), max(total)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    if case["op"] == "sample":
        st = _prepare_sample(case, gen)
    else:
        st, rows, longest, furthest = _prepare_cache(case, gen)
        heads, kv, d = case["heads"], case["kv_heads"], case["head_dim"]
        st.update(rows=rows, longest=longest, furthest=furthest)
        if case["op"] == "append":
            st["qkv"] = _values(case, gen, rows, (heads + 2 * kv) * d)
            half = case["rotary"] // 2
            angle = torch.arange(furthest, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
            st["cos"], st["sin"] = angle.cos().float(), angle.sin().float()
            st["q"] = torch.zeros(rows, heads * d, dtype=st["qkv"].dtype, device="cuda")
        else:
            st["q"] = _values(case, gen, rows, heads * d) * 1.5
            st["out"] = torch.zeros_like(st["q"])
    st["case"] = case
    if own:
        st["handles"] = _handles(st)
    return st


# ------------------------------------------------------------------------------------------------ the framework's calls

_backend = None


def _handles(st):
    """What a program that serves with the framework keeps from call to call: the buffer handles, the argument block, the workspace."""
    global _backend
    from fandhe_ai_b200 import BF16, F32, Backend
    from fandhe_ai_b200 import paged_kv as P
    from fandhe_ai_b200.decoder import SampleArgs

    if _backend is None:
        _backend = Backend(0)
    be, case = _backend, st["case"]
    h = {k: be.import_tensor(t) for k, t in st.items() if isinstance(t, torch.Tensor)}
    dtype = F32 if case["dtype"] == "f32" else BF16
    if case["op"] == "sample":
        h["args"] = SampleArgs(rows=case["rows"], vocab=case["vocab"], row_stride=case["stride"], dtype=dtype)
        return h
    blocks, block, width = st["k_pool"].shape
    layout = P.PagedKvLayout(blocks, block, width, BF16)
    common = dict(layout=layout, batch=case["seqs"], rows=st["rows"], num_heads=case["heads"], num_kv_heads=case["kv_heads"],
                  max_blocks_per_seq=st["tables"].shape[1], io_dtype=dtype)
    if case["op"] == "append":
        h["args"] = P.RopeAppendArgs(rotary_dim=case["rotary"], adjacent_pairs=case["pairs"] == "adjacent", n_positions=st["cos"].shape[0], **common)
    else:
        h["args"] = P.PagedChunkArgs(max_q_len=st["longest"], max_seq_len=st["furthest"], scale=case["head_dim"] ** -0.5, **common)
        h["workspace"] = be.import_tensor(torch.zeros(max(16, P.paged_chunk_workspace(be, h["args"])), dtype=torch.uint8, device="cuda"))
    return h


def _own(st):
    from fandhe_ai_b200 import paged_kv as P
    from fandhe_ai_b200.decoder import sample_tokens

    h, op = st["handles"], st["case"]["op"]
    if op == "sample":
        sample_tokens(_backend, h["logits"], h["args"], h["u"], h["ids"], temperature=h["temperature"], top_k=h["top_k"], top_p=h["top_p"],
                      min_p=h["min_p"], prob=h["prob"], kept=h["kept"])
        return dict(ids=st["ids"], prob=st["prob"], kept=st["kept"])
    if op == "append":
        P.rope_paged_kv_append(_backend, h["qkv"], h["cos"], h["sin"], h["tables"], h["q_starts"], h["seq_lens"], h["k_pool"], h["v_pool"],
                               h["args"], h["q"])
        return dict(q=st["q"], k_pool=st["k_pool"], v_pool=st["v_pool"])
    P.paged_chunk_attention(_backend, h["q"], h["k_pool"], h["v_pool"], h["tables"], h["q_starts"], h["seq_lens"], h["args"], h["workspace"],
                            h["out"])
    return dict(out=st["out"])


# ------------------------------------------------------------------------------------------------ the plain forms


def _plain_append(st):
    case = st["case"]
    heads, kv, d, block, rot = (case[k] for k in ("heads", "kv_heads", "head_dim", "block", "rotary"))
    row = torch.arange(st["rows"], device="cuda")
    starts = st["q_starts"].long()
    seq = torch.searchsorted(starts, row, right=True) - 1
    pos = st["seq_lens"].long()[seq] - (starts[seq + 1] - row)
    slot = st["tables"].long()[seq, pos // block] * block + pos % block
    x = st["qkv"].float().view(st["rows"], heads + 2 * kv, d)
    cos, sin = st["cos"][pos][:, None], st["sin"][pos][:, None]
    turned = x[:, :heads + kv].clone()
    if case["pairs"] == "half":
        a, b = x[:, :heads + kv, :rot // 2], x[:, :heads + kv, rot // 2:rot]
        turned[:, :, :rot // 2], turned[:, :, rot // 2:rot] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[:, :heads + kv, 0:rot:2], x[:, :heads + kv, 1:rot:2]
        turned[:, :, 0:rot:2], turned[:, :, 1:rot:2] = a * cos - b * sin, b * cos + a * sin
    st["q"].copy_(turned[:, :heads].reshape(st["rows"], -1))
    st["k_pool"].view(-1, kv * d)[slot] = turned[:, heads:].reshape(st["rows"], -1).to(st["k_pool"].dtype)
    st["v_pool"].view(-1, kv * d)[slot] = x[:, heads + kv:].reshape(st["rows"], -1).to(st["v_pool"].dtype)
    return dict(q=st["q"], k_pool=st["k_pool"], v_pool=st["v_pool"])


def _plain_attention(st):
    case = st["case"]
    heads, kv, d, block = (case[k] for k in ("heads", "kv_heads", "head_dim", "block"))
    batch, group, most, far = case["seqs"], heads // kv, st["longest"], st["furthest"]
    starts, total = st["q_starts"].long(), st["seq_lens"].long()
    new = starts[1:] - starts[:-1]
    i, j = torch.arange(most, device="cuda"), torch.arange(far, device="cuda")
    real = i < new[:, None]
    cached = j < total[:, None]
    slot = torch.where(cached, st["tables"].long()[:, j // block] * block + j % block, 0)
    k = st["k_pool"].view(-1, kv, d)[slot].float().permute(0, 2, 3, 1)
    v = torch.where(cached[:, :, None, None], st["v_pool"].view(-1, kv, d)[slot].float(), 0.0).permute(0, 2, 1, 3)
    row = torch.where(real, starts[:-1, None] + i, 0)
    q = st["q"].float().view(-1, kv, group, d)[row].permute(0, 2, 1, 3, 4).reshape(batch, kv, most * group, d)
    s = (torch.matmul(q, k) * d ** -0.5).view(batch, kv, most, group, far)
    s.masked_fill_((j > (total - new)[:, None, None] + i[:, None])[:, None, :, None], -math.inf)
    s.sub_(s.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(s.view(batch, kv, most * group, far), v).view(batch, kv, most, group, d) / s.sum(-1, keepdim=True)
    out = st["out"]
    out[row[real]] = o.permute(0, 2, 1, 3, 4).reshape(batch, most, heads * d)[real].to(out.dtype)
    return dict(out=out)


def _plain_sample(st):
    """Softmax weights under the row's temperature; the kept tokens are the first ones in the order of falling logits (equal logits: the lower
    index first) that top-k, then top-p over what top-k leaves, then min-p against the largest weight allow; the draw is the first kept index
    at which the running sum passes u times the sum.  In 64 bits: tokens stand next to the borders of these sums."""
    x = st["logits"][:, :st["case"]["vocab"]].double()
    n = x.shape[1]
    t, p, m, u = (st[k].double()[:, None] for k in ("temperature", "top_p", "min_p", "u"))
    k = torch.where(st["top_k"] > 0, st["top_k"], n)[:, None]
    w = ((x - x.amax(1, keepdim=True)) / t).exp()
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    rank = torch.arange(n, device="cuda")[None]
    ws = torch.where(rank < k, w.gather(1, order), 0.0)
    run_ = ws.cumsum(1)
    before = torch.cat([torch.zeros_like(run_[:, :1]), run_[:, :-1]], 1)
    keep = (ws > 0) & ((before < p * run_[:, -1:]) | (p >= 1)) & (ws >= m)
    keep |= rank == 0
    kept = torch.zeros_like(w).scatter_(1, order, torch.where(keep, ws, 0.0))
    c = kept.cumsum(1)
    ids = (c <= u * c[:, -1:]).sum(1)
    return dict(ids=ids.to(torch.int32), prob=(kept.gather(1, ids[:, None]) / c[:, -1:])[:, 0].float(), kept=keep.sum(1).to(torch.int32))


def run(state):
    if own:
        # the framework works on its context's stream, the tensors belong to torch's: in order on the device, without the host waiting
        stream = torch.cuda.current_stream().cuda_stream
        _backend.wait_stream(stream)
        out = _own(state)
        _backend.stream_wait(stream)
        return out
    return {"append": _plain_append, "attention": _plain_attention, "sample": _plain_sample}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------------ 64 bits


def _exact_append(case, st):
    new, total = _lengths(case)
    heads, kv, d, block, rot = (case[k] for k in ("heads", "kv_heads", "head_dim", "block", "rotary"))
    pos = torch.cat([torch.arange(t - n, t) for n, t in zip(new, total)])
    tab = st["tables"].cpu().long()
    slots = torch.cat([tab[b, torch.arange(t - n, t) // block] * block + torch.arange(t - n, t) % block for b, (n, t) in enumerate(zip(new, total))])
    qkv = st["qkv"].cpu().double().view(-1, heads + 2 * kv, d)
    z = torch.complex(st["cos"].cpu().double(), st["sin"].cpu().double())[pos][:, None, :]
    first = torch.arange(rot // 2) if case["pairs"] == "half" else torch.arange(0, rot, 2)
    second = first + (rot // 2 if case["pairs"] == "half" else 1)
    qk = qkv[:, :heads + kv]
    turn = torch.complex(qk[:, :, first], qk[:, :, second]) * z
    qk[:, :, first], qk[:, :, second] = turn.real, turn.imag
    pools = {}
    for name, rows in (("k_pool", qk[:, heads:]), ("v_pool", qkv[:, heads + kv:])):
        pool = st[name].cpu().double().view(-1, kv * d)
        pool[slots] = rows.reshape(-1, kv * d)
        pools[name] = pool.view(st[name].shape)
    return dict(q=qk[:, :heads].reshape(-1, heads * d), **pools)


def _exact_attention(case, st):
    new, total = _lengths(case)
    heads, kv, d, block = (case[k] for k in ("heads", "kv_heads", "head_dim", "block"))
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for b, (n, t) in enumerate(zip(new, total)):
        blocks = st["tables"][b, :-(-t // block)].long()
        ks, vs = (st[name][blocks].reshape(-1, kv, d)[:t].double() for name in ("k_pool", "v_pool"))
        q = st["q"][at:at + n].double().view(n, kv, heads // kv, d)
        seen = torch.arange(t, device="cuda")[None, :] <= torch.arange(t - n, t, device="cuda")[:, None]
        for h in range(kv):
            a = torch.einsum("igd,jd->gij", q[:, h], ks[:, h]) / math.sqrt(d)
            a = torch.softmax(a.masked_fill(~seen, -math.inf), -1)
            out[at:at + n].view(n, kv, heads // kv, d)[:, h] = torch.einsum("gij,jd->igd", a, vs[:, h])
        at += n
    return dict(out=out)


def _exact_sample(case, st):
    x = st["logits"][:, :case["vocab"]].double().cpu().numpy()
    t, k, p, m, u = (st[n].double().cpu().numpy() for n in ("temperature", "top_k", "top_p", "min_p", "u"))
    prob = np.zeros(len(x))
    for r, row in enumerate(x):
        live = np.flatnonzero(row > -np.inf)
        live = live[np.lexsort((live, -row[live]))]
        if k[r] > 0:
            live = live[:int(k[r])]
        w = np.exp((row[live] - row[live[0]]) / t[r])
        if p[r] < 1:
            n = int(np.searchsorted(np.cumsum(w), p[r] * w.sum())) + 1
            live, w = live[:n], w[:n]
        n = max(1, int((w >= m[r]).sum()))
        live, w = live[:n], w[:n]
        w = w[np.argsort(live)]
        prob[r] = w[min(int(np.searchsorted(np.cumsum(w), u[r] * w.sum(), side="right")), len(w) - 1)] / w.sum()
    return dict(ids=None, prob=prob, kept=None)   # whole numbers: the plain form's own


def exact(case, seed):
    st = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "sample": _exact_sample}[case["op"]](case, st)
