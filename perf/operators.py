"""Operators for language-model training and serving around the attention kernels, as measurable cases.

  ranges     which keys each query sees, built on the GPU from lengths: documents packed into a row, a prefix every row of
             a document sees, a sliding window, ragged caches.  Row i of a batch entry sees keys [first, end)
  rotary     q and k rotated by their positions; a training step returns the rotated tensors and both gradients
  attention  softmax(cap tanh(scale q.k / cap) - slope_h |position - key|) v over each row's keys: a training step with every
             gradient, or a forward without gradients (a prompt's chunk, one new token for each running request)

A row that sees no key has an output of zeros.
"""
import os
import sys

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
# What a drawn attention case may cost: query-key pairs of all heads, times the head size (train_documents_bf16 has 1.1e10)
MOST_PAIRS_D = 1.0e10
MOST_ROTARY = 8.0e7


def _fa():
    folder = os.path.join(os.getcwd(), "flash-attn-v100_b200")      # the package lies below the repository's root
    if folder not in sys.path:
        sys.path.insert(0, folder)
    import flash_attention_v100
    return flash_attention_v100


# ---------------------------------------------------------------------------------------------------------- the cases
def _ranges(name, B, Nq, Nk, causal=True, docs=0, prefix=0, window=0, cache=False):
    """docs: documents a row is cut into (0: none); prefix: longest visible prefix of a document; window: keys back;
    cache: each batch entry has its own number of keys, its queries are the last Nq of them."""
    case = {"op": "ranges", "B": B, "Nq": Nq, "Nk": Nk, "causal": causal, "docs": docs, "prefix": prefix,
            "window": window, "cache": cache}
    return dict(case, name=name) if name else case


def _rotary(name, B, N, H, Hkv, D, rotary_dim, dtype, interleaved, train, far=0, factor=1.0):
    """far: the largest first position of a batch entry; factor: attention factor of a scaled long-context table."""
    case = {"op": "rotary", "B": B, "N": N, "H": H, "Hkv": Hkv, "D": D, "rotary_dim": rotary_dim, "dtype": dtype,
            "interleaved": interleaved, "train": train, "far": far, "factor": factor}
    return dict(case, name=name) if name else case


def _attention(name, B, Nq, Nk, H, Hkv, D, dtype, train, causal=True, docs=0, prefix=0, window=0, cache=False, cap=0.0, slopes=False):
    case = {"op": "attention", "B": B, "Nq": Nq, "Nk": Nk, "H": H, "Hkv": Hkv, "D": D, "dtype": dtype, "train": train, "causal": causal,
            "docs": docs, "prefix": prefix, "window": window, "cache": cache, "cap": cap, "slopes": slopes}
    return dict(case, name=name) if name else case


def listed():
    return [
        # the plan of one decoding step: a row for each of 64 running requests
        _ranges("ranges_decode_b64", 64, 1, 8192, cache=True, window=4096),
        # the plan of a training step: 32 documents of any length in every row of 16384 tokens, prefixes visible
        _ranges("ranges_documents_b8_n16384", 8, 16384, 16384, docs=32, prefix=500),
        # one new token for each of 32 requests, far into their contexts: launch latency
        _rotary("rotary_decode_b32", 32, 1, 32, 8, 128, 128, "bf16", False, False, far=100000, factor=1.1),
        # interleaved pairs, a part of an odd-sized head, odd lengths
        _rotary("rotary_part_fp16_n1021", 3, 1021, 12, 12, 80, 32, "fp16", True, True, far=5000),
        # a training step's q and k, grouped heads
        _rotary("rotary_train_b4_n4096", 4, 4096, 32, 8, 128, 128, "bf16", False, True),
        # one request, one token, a short cache: latency
        _attention("decode_b1_n33", 1, 1, 33, 8, 8, 64, "fp16", False, cache=True, cap=20.0),
        # one new token for each of 32 requests of their own lengths, capped scores and distances: a read of the caches
        _attention("decode_b32_n8192", 32, 1, 8192, 32, 8, 128, "bf16", False, cache=True, cap=30.0, slopes=True),
        # the next chunk of a long prompt in a sliding window, odd lengths
        _attention("chunk_n700_k8892", 1, 700, 8892, 32, 8, 128, "bf16", False, cache=True, window=4096, cap=50.0),
        # training with distances only, head size between the powers of two, odd length
        _attention("train_distance_fp16_n1021", 4, 1021, 1021, 12, 12, 80, "fp16", True, slopes=True),
        # fp32 training on short packed rows whose last documents end before the row does
        _attention("train_fp32_n500", 2, 500, 500, 4, 4, 64, "fp32", True, docs=5, cap=15.0, slopes=True),
        # training on packed documents with a visible prefix, capped scores, grouped heads
        _attention("train_prefix_cap_bf16", 4, 2048, 2048, 16, 4, 64, "bf16", True, docs=3, prefix=300, cap=30.0),
        # the ordinary training step on packed documents
        _attention("train_documents_bf16", 4, 4096, 4096, 32, 32, 128, "bf16", True, docs=8),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["ranges", "rotary", "attention", "attention", "attention"])
    if op == "ranges":
        kind = rng.choice(["cache", "docs", "docs", "window"])
        if kind == "cache":
            return _ranges(None, _log(rng, 2, 256), rng.choice([1, 1, 1, 4]), _log(rng, 257, 16384), cache=True, window=rng.choice([0, _log(rng, 16, 4096)]))
        N = _log(rng, 129, 16384)
        B, docs = rng.randint(1, 8), rng.randint(3, 32)
        if kind == "docs":
            causal = rng.random() < 0.7
            return _ranges(None, B, N, N, causal=causal, docs=docs, prefix=rng.choice([0, _log(rng, 1, 600)]) if causal else 0)
        return _ranges(None, B, N, N, causal=rng.random() < 0.5, docs=docs, window=_log(rng, 1, N))
    if op == "rotary":
        D = rng.choice([64, 80, 96, 128, 128])
        Hkv = rng.choice([1, 4, 8, 12])
        H = Hkv * rng.choice([1, 2, 4])
        B = _log(rng, 1, 32)
        N = min(_log(rng, 1, 8192), max(1, int(MOST_ROTARY / (B * (H + Hkv) * D))))
        rd = rng.choice([D, D, D // 2, 32])
        return _rotary(None, B, N, H, Hkv, D, rd, rng.choice(["bf16", "bf16", "fp16", "fp32"]), rng.random() < 0.4, rng.random() < 0.5,
                       far=rng.choice([0, 0, 5000, 100000]), factor=rng.choice([1.0, 1.1]))
    D = rng.choice([64, 64, 80, 128, 128, 128])
    Hkv = rng.choice([2, 4, 8])
    H = Hkv * rng.choice([1, 2, 4])
    cap = rng.choice([0.0, 15.0, 30.0, 50.0])
    slopes = rng.random() < 0.4
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp16"])
    if rng.random() < 0.4:
        Nk = _log(rng, 33, 16384)
        if rng.random() < 0.7:
            Nq, B = 1, _log(rng, 1, 64)
        else:
            Nq, B = min(Nk, _log(rng, 2, 1024)), rng.randint(1, 3)
        window = rng.choice([0, 0, _log(rng, 16, 4096)])
        return _attention(None, B, Nq, Nk, H, Hkv, D, dtype, False, cache=True, window=window, cap=cap, slopes=slopes)
    if rng.random() < 0.1:
        return _attention(None, rng.randint(1, 2), _log(rng, 17, 700), 0, 4, 4, rng.choice([32, 64]), "fp32", True, docs=rng.randint(1, 5), cap=cap, slopes=slopes)
    N = _log(rng, 65, 8192)
    while N * N * H * D > 4 * MOST_PAIRS_D:
        N = N * 3 // 4 | 1
    B = rng.randint(1, max(1, min(8, int(4 * MOST_PAIRS_D / (N * N * H * D)))))
    causal = rng.random() < 0.8
    docs = rng.choice([0, 1, 3, 8])
    window = _log(rng, 16, 4096) if docs == 0 and rng.random() < 0.5 else 0
    prefix = _log(rng, 1, 400) if docs and causal and rng.random() < 0.4 else 0
    return _attention(None, B, N, N, H, Hkv, D, dtype, rng.random() < 0.8, causal=causal, docs=docs, prefix=prefix, window=window, cap=cap, slopes=slopes)


# ---------------------------------------------------------------------------------------------------------- the inputs
def _plan_inputs(case, g, dev):
    """What the ranges are built from: offsets (B, docs + 1), prefixes (B, docs), key counts and first positions (B,)."""
    B, Nq, Nk = case["B"], case["Nq"], case["Nk"] or case["Nq"]
    state = {"offsets": None, "prefixes": None, "counts": None, "first_positions": None}
    if case["docs"]:
        # documents of any length; together they fill nine tenths of the row or more, what is behind them is padding
        cuts = torch.rand(B, case["docs"] - 1, generator=g).sort(dim=1).values
        total = torch.randint(Nq - Nq // 10, Nq + 1, (B, 1), generator=g)
        inner = (cuts * total).to(torch.int64)
        state["offsets"] = torch.cat([torch.zeros(B, 1, dtype=torch.int64), inner, total], dim=1).to(torch.int32).to(dev)
        if case["prefix"]:
            state["prefixes"] = torch.randint(0, case["prefix"] + 1, (B, case["docs"]), generator=g).to(torch.int32).to(dev)
    if case["cache"]:
        counts = torch.randint(max(Nq, Nk // 4), Nk + 1, (B,), generator=g)
        if case["op"] == "attention":
            counts[0] = Nk
        state["counts"] = counts.to(torch.int32).to(dev)
        state["first_positions"] = (counts - Nq).to(torch.int32).to(dev)
    return state


def _build(case, state):
    """The framework's ranges for these inputs."""
    return _fa().build_key_ranges(case["Nq"], case["Nk"] or case["Nq"], batch=case["B"], causal=case["causal"], window=case["window"] or None,
                                  document_offsets=state["offsets"], prefix_lengths=state["prefixes"], key_lengths=state["counts"],
                                  query_offsets=state["first_positions"], device=state["device"])


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator().manual_seed(seed)
    gd = torch.Generator(device=dev).manual_seed(seed)
    state = {"case": case, "device": dev}
    if case["op"] == "ranges":
        state.update(_plan_inputs(case, g, dev))
        return state
    dtype = DTYPES[case["dtype"]]
    B, H, Hkv, D = case["B"], case["H"], case["Hkv"], case["D"]

    def normal(n, heads, std=1.0):
        return (torch.randn(B, n, heads, D, generator=gd, device=dev) * std).to(dtype)

    if case["op"] == "rotary":
        N = case["N"]
        state["q"], state["k"] = normal(N, H), normal(N, Hkv)
        if case["train"]:
            state["dq"], state["dk"] = normal(N, H, 0.01), normal(N, Hkv, 0.01)
            state["q"].requires_grad_(True)
            state["k"].requires_grad_(True)
        first = torch.randint(0, case["far"] + 1, (B, 1), generator=g)
        state["positions"] = (first + torch.arange(N)).to(torch.int32).to(dev)
        # the table a program keeps: one frequency for each pair, in 64 bits (positions are far, angles large)
        half = case["rotary_dim"] // 2
        state["inv_freq"] = (10000.0 ** (-torch.arange(half, dtype=torch.float64) / half)).to(dev)
        return state
    Nq, Nk = case["Nq"], case["Nk"] or case["Nq"]
    # scores of a few units, so that a cap bends them
    state["q"], state["k"], state["v"] = normal(Nq, H, 2.5), normal(Nk, Hkv), normal(Nk, Hkv)
    if case["train"]:
        state["do"] = normal(Nq, H)
        for n in "qkv":
            state[n].requires_grad_(True)
    state["slopes"] = (2.0 ** (-8.0 * torch.arange(1, H + 1, dtype=torch.float32) / H)).to(dev) if case["slopes"] else None
    state.update(_plan_inputs(case, g, dev))
    if own:
        state["ranges"] = _build(case, state)       # built once for a step, read by every layer
    else:
        state["rows"] = _rows_plain(case, state)
    return state


# ---------------------------------------------------------------------------------------------------- the plain forms
def _rows_plain(case, state):
    """first, end, position within the document: (B, Nq) whole numbers."""
    dev = state["device"]
    B, Nq, Nk = case["B"], case["Nq"], case["Nk"] or case["Nq"]
    at = torch.arange(Nq, device=dev).expand(B, Nq)
    if state["first_positions"] is not None:
        at = at + state["first_positions"].long()[:, None]
    start = torch.zeros_like(at)
    end = torch.full_like(at, Nk)
    if state["counts"] is not None:
        end = torch.minimum(end, state["counts"].long()[:, None])
    prefix = torch.zeros_like(at)
    inside = torch.ones_like(at, dtype=torch.bool)
    if state["offsets"] is not None:
        off = state["offsets"].long()
        passed = (off[:, None, :] <= at[:, :, None]).sum(dim=2)               # boundaries at or before the row
        inside = (passed > 0) & (passed < off.shape[1])
        m = (passed - 1).clamp(0, off.shape[1] - 2)
        start = torch.where(inside, off.gather(1, m), start)
        end = torch.minimum(end, off.gather(1, m + 1))
        if state["prefixes"] is not None:
            prefix = state["prefixes"].long().gather(1, m)
    first = start
    if case["window"]:
        first = torch.maximum(first, at - case["window"] + 1)
        if not case["causal"]:
            end = torch.minimum(end, at + case["window"])
    if case["causal"]:
        end = torch.minimum(end, torch.maximum(at + 1, torch.where(prefix > 0, start + prefix, torch.zeros_like(at))))
    seen = inside & (first < end)
    zero = torch.zeros_like(at)
    return (torch.where(seen, first, zero).int(), torch.where(seen, end, zero).int(), torch.where(inside, at - start, zero).int())


def _rotate_plain(x, cos, sin, half, interleaved):
    part = x[..., :2 * half].float()
    if interleaved:
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = part[..., :half], part[..., half:]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned.to(x.dtype), x[..., 2 * half:]), dim=-1)


def _rotary_plain(state):
    case = state["case"]
    half = case["rotary_dim"] // 2
    angle = state["positions"].double()[:, :, None, None] * state["inv_freq"]
    cos, sin = (angle.cos() * case["factor"]).float(), (angle.sin() * case["factor"]).float()
    with torch.no_grad():
        out = [_rotate_plain(state[n], cos, sin, half, case["interleaved"]) for n in ("q", "k")]
        if case["train"]:
            out += [_rotate_plain(state[n], cos, -sin, half, case["interleaved"]) for n in ("dq", "dk")]
    return tuple(out)


def _attention_plain(state):
    case = state["case"]
    H, Hkv, D = case["H"], case["Hkv"], case["D"]
    group, scale, cap = H // Hkv, D ** -0.5, case["cap"]
    first, end, _ = state["rows"]
    q, k, v = (state[n].detach() for n in "qkv")
    train = case["train"]
    Nq, Nk = q.shape[1], k.shape[1]
    key = torch.arange(Nk, device=q.device)
    at = torch.arange(Nq, device=q.device).expand(q.shape[0], Nq)
    if state["first_positions"] is not None:
        at = at + state["first_positions"].long()[:, None]
    o = torch.empty_like(q)
    if train:
        dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    for b in range(q.shape[0]):                       # one batch entry at a time: its scores are all there at once
        hidden = (key < first[b][:, None]) | (key >= end[b][:, None])
        distance = (at[b][:, None] - key).abs().float()
        qf = q[b].float().transpose(0, 1).reshape(Hkv, group * Nq, D)              # heads of a K/V head together
        kf, vf = (t[b].float().transpose(0, 1) for t in (k, v))
        s = torch.matmul(qf, kf.transpose(1, 2)).mul_(scale).view(H, Nq, Nk)
        bend = None
        if cap:
            bend = torch.tanh(s.div_(cap))
            s = bend * cap
        if state["slopes"] is not None:
            s = s - state["slopes"][:, None, None] * distance
        s = s.masked_fill_(hidden, float("-inf"))
        top = s.amax(dim=2, keepdim=True)
        p = torch.exp(s.sub_(top.masked_fill(top == float("-inf"), 0.0)))
        total = p.sum(dim=2, keepdim=True)
        p = p.div_(total.masked_fill(total == 0.0, 1.0)).view(Hkv, group * Nq, Nk)
        of = torch.matmul(p, vf)
        o[b] = of.view(H, Nq, D).transpose(0, 1).to(o.dtype)
        if not train:
            continue
        gf = state["do"][b].float().transpose(0, 1).reshape(Hkv, group * Nq, D)
        dv[b] = torch.matmul(p.transpose(1, 2), gf).transpose(0, 1).to(dv.dtype)
        ds = torch.matmul(gf, vf.transpose(1, 2)).sub_((gf * of).sum(dim=2, keepdim=True)).mul_(p)
        if cap:
            ds = ds.mul_(1.0 - bend.square_().view_as(ds))
        ds = ds.mul_(scale)
        dq[b] = torch.matmul(ds, kf).view(H, Nq, D).transpose(0, 1).to(dq.dtype)
        dk[b] = torch.matmul(ds.transpose(1, 2), qf).transpose(0, 1).to(dk.dtype)
    return (o, dq, dk, dv) if train else (o,)


# ------------------------------------------------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    if not own:
        if case["op"] == "ranges":
            return _rows_plain(case, state)
        return _rotary_plain(state) if case["op"] == "rotary" else _attention_plain(state)
    fa = _fa()
    if case["op"] == "ranges":
        ranges = _build(case, state)
        return ranges.first, ranges.end, ranges.positions
    if case["op"] == "rotary":
        q, k = state["q"], state["k"]
        y = fa.rotary_embedding(q, k, positions=state["positions"], inv_freq=state["inv_freq"], interleaved=case["interleaved"],
                                attention_factor=case["factor"])
        if not case["train"]:
            return y
        return tuple(t.detach() for t in y) + torch.autograd.grad(y, (q, k), (state["dq"], state["dk"]))
    q, k, v = state["q"], state["k"], state["v"]
    o = fa.flash_attention_v100_with_rules(q, k, v, score_cap=case["cap"] or None, distance_slopes=state["slopes"], key_ranges=state["ranges"])
    if not case["train"]:
        return (o,)
    return (o.detach(),) + torch.autograd.grad(o, (q, k, v), state["do"])


# ------------------------------------------------------------------------------------------ the definition, in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "ranges":
        return None                                 # whole numbers
    if case["op"] == "rotary":
        angle = state["positions"].double().unsqueeze(2) * state["inv_freq"].view(1, 1, -1)
        turn = torch.polar(torch.full_like(angle, case["factor"]), angle).unsqueeze(2)         # a complex number for each pair
        half = case["rotary_dim"] // 2

        def rotated(x, by):
            x = x.detach().double()
            head, rest = x[..., :2 * half], x[..., 2 * half:]
            if case["interleaved"]:
                z = torch.view_as_complex(head.unflatten(-1, (half, 2)).contiguous()) * by
                y = torch.view_as_real(z).flatten(-2)
            else:
                z = torch.complex(head[..., :half], head[..., half:]) * by
                y = torch.cat((z.real, z.imag), dim=-1)
            return torch.cat((y, rest), dim=-1)

        out = [rotated(state["q"], turn), rotated(state["k"], turn)]
        if case["train"]:
            out += [rotated(state["dq"], turn.conj()), rotated(state["dk"], turn.conj())]
        return tuple(out)
    B, H, D = case["B"], case["H"], case["D"]
    group = H // case["Hkv"]
    Nq, Nk = case["Nq"], case["Nk"] or case["Nq"]
    if B * H * Nq * Nk * D * (2.5 if case["train"] else 1) > 3e12:
        return None                                 # (in 64 bits some twenty seconds)
    dev = state["device"]
    outs = [torch.empty(B, Nq, H, D, dtype=torch.float64, device=dev)]
    if case["train"]:
        outs += [torch.empty(B, Nq, H, D, dtype=torch.float64, device=dev)] + [torch.zeros(B, Nk, case["Hkv"], D, dtype=torch.float64, device=dev) for _ in "kv"]
    i, j = torch.arange(Nq, device=dev).view(-1, 1), torch.arange(Nk, device=dev).view(1, -1)
    for b in range(B):
        # the mask from its definition, pair by pair
        t = i + (0 if state["first_positions"] is None else int(state["first_positions"][b]))
        sees = (j < (Nk if state["counts"] is None else int(state["counts"][b]))) & (t >= 0)
        prefixed = torch.zeros_like(sees)
        if state["offsets"] is not None:
            off = state["offsets"][b].tolist()
            same = torch.zeros(Nq, Nk, dtype=torch.bool, device=dev)
            for m in range(len(off) - 1):
                rows, cols = (t >= off[m]) & (t < off[m + 1]), (j >= off[m]) & (j < off[m + 1])
                same |= rows & cols
                if state["prefixes"] is not None:
                    prefixed = prefixed | (rows & cols & (j < off[m] + int(state["prefixes"][b, m])))
            sees = sees & same
        if case["window"]:
            sees = sees & (t - j < case["window"]) & (j - t < case["window"])
        if case["causal"]:
            sees = sees & ((j <= t) | prefixed)
        none = ~sees.any(dim=1, keepdim=True)
        for h in range(H):
            q, k, v = state["q"][b, :, h].detach().double(), state["k"][b, :, h // group].detach().double(), state["v"][b, :, h // group].detach().double()
            x = q @ k.T / D ** 0.5
            slope_of_cap = 1.0
            if case["cap"]:
                bent = torch.tanh(x / case["cap"])
                x, slope_of_cap = case["cap"] * bent, 1.0 - bent * bent
            if state["slopes"] is not None:
                x = x - float(state["slopes"][h]) * (t - j).abs().double()
            x = torch.where(sees, x, torch.full_like(x, float("-inf")))
            p = torch.where(none, torch.zeros_like(x), torch.softmax(torch.where(none, torch.zeros_like(x), x), dim=1))
            o = p @ v
            outs[0][b, :, h] = o
            if case["train"]:
                do = state["do"][b, :, h].double()
                outs[3][b, :, h // group] += p.T @ do
                dp = do @ v.T
                dx = p * (dp - (p * dp).sum(dim=1, keepdim=True)) * slope_of_cap / D ** 0.5
                outs[1][b, :, h] = dx @ k
                outs[2][b, :, h // group] += dx.T @ q
    return tuple(outs)


# ------------------------------------------------------------------------------------------------- what cannot be saved
def _pairs(case):
    """Query-key pairs of one head of one batch entry, on average over what the inputs may be."""
    Nq, Nk = case["Nq"], case["Nk"] or case["Nq"]
    if case["docs"]:
        n = 0.95 * Nq                               # what the documents fill
        m = case["docs"]
        square = n * n * 2.0 / (m + 1)              # sum of the squares of m uneven parts
        if not case["causal"]:
            return square
        return min(square, square / 2 + (case["prefix"] / 2) ** 2 / 2 * m)
    keys = Nk
    if case["cache"]:
        keys = Nk if case["B"] == 1 else Nk * (1 + (case["B"] - 1) * 0.625) / case["B"]
    if case["window"]:
        w = min(case["window"], Nk)
        return Nq * min(w, keys) if case["causal"] else Nq * min(2 * w, keys)
    return Nq * (keys - Nq / 2) if case["causal"] else Nq * keys


def work(case):
    if case["op"] == "ranges":
        rows = case["B"] * case["Nq"]
        return {"bytes": 12 * rows + 8 * case["B"] * (case["docs"] + 2), "flops": 8 * rows}
    size = DTYPES[case["dtype"]].itemsize
    B, H, Hkv, D = case["B"], case["H"], case["Hkv"], case["D"]
    if case["op"] == "rotary":
        n = B * case["N"] * (H + Hkv) * D
        passes = 2 if case["train"] else 1
        return {"bytes": passes * (2 * n * size + 4 * B * case["N"]), "flops": passes * 3 * n * case["rotary_dim"] // D}
    Nq, Nk = case["Nq"], case["Nk"] or case["Nq"]
    pairs = _pairs(case)
    keys = min(Nk, pairs / Nq + Nq) if case["cache"] else Nk
    q_bytes, k_bytes = B * Nq * H * D * size, B * keys * Hkv * D * size
    if not case["train"]:
        return {"bytes": int(2 * q_bytes + 2 * k_bytes), "flops": int(4 * B * H * pairs * D)}
    return {"bytes": int(4 * q_bytes + 4 * k_bytes), "flops": int(14 * B * H * pairs * D)}
