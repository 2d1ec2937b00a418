"""Workloads of the paged 8-bit key/value cache: append, attend, copy_pages.

A cache layer is a pool of pages ``codes[page, K or V, kv head, slot, d]`` in
e4m3 with one power-of-two scale ``2 ** exps[page, K or V, kv head]`` for each
page, side and head.  A sequence is a row of page numbers and a length; its
new tokens are the last ones of that length.  Each case below is one call of
one operator; ``run`` computes it in elementary torch operations, or with
``own`` set by the framework's kernels.
"""

import random
import sys
from pathlib import Path

import numpy as np
import torch

own = False

E_MIN, E_MAX = -32, 63          # range of a page's exponent
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------


def _attend(name, seqs, kv, q, heads, kv_heads, head_dim, page=64, dtype="bf16", window=0, sinks=0):
    return {"name": name, "op": "attend", "seqs": seqs, "kv_min": kv[0], "kv_max": kv[1],
            "q_min": q[0], "q_max": q[1], "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "page": page, "dtype": dtype, "window": window, "sinks": sinks}


def _append(name, seqs, kv, q, kv_heads, head_dim, page=64, dtype="bf16"):
    return {"name": name, "op": "append", "seqs": seqs, "kv_min": kv[0], "kv_max": kv[1],
            "q_min": q[0], "q_max": q[1], "kv_heads": kv_heads, "head_dim": head_dim,
            "page": page, "dtype": dtype}


def _copy(name, layers, pages, pairs, kv_heads, head_dim, page=64):
    return {"name": name, "op": "copy", "layers": layers, "pages": pages, "pairs": pairs,
            "kv_heads": kv_heads, "head_dim": head_dim, "page": page}


def listed():
    return [
        # one conversation, one new token: latency
        _attend("decode_one", 1, (1025, 1025), (1, 1), 32, 8, 128),
        # a full server: one new token for each of 64 conversations of mixed length
        _attend("decode_batch", 64, (700, 8191), (1, 1), 32, 8, 128),
        # two very long documents and few kv heads: the work has to be split over the keys
        _attend("decode_long", 2, (131071, 131071), (1, 1), 16, 2, 128, page=128, dtype="f16"),
        # a layer with a sliding window and four first tokens that stay visible
        _attend("decode_window", 48, (5000, 32767), (1, 1), 64, 8, 64, window=1024, sinks=4),
        # five draft tokens of each conversation checked at once
        _attend("verify_drafts", 16, (500, 6000), (5, 5), 20, 5, 128),
        # chunks of several prompts behind histories of their own, in one call
        _attend("prompt_chunks", 6, (1500, 4000), (200, 1500), 32, 8, 128),
        # one long prompt from its first token
        _attend("prompt_long", 1, (8191, 8191), (8191, 8191), 32, 8, 128),
        # a long prompt through a layer with a sliding window
        _attend("prompt_window", 1, (8191, 8191), (8191, 8191), 64, 8, 64, dtype="f16", window=512, sinks=4),
        # one new token for each of 64 conversations
        _append("append_decode", 64, (700, 8191), (1, 1), 8, 128),
        # several prompts at once
        _append("append_prompts", 6, (6000, 9000), (3000, 8000), 8, 128),
        # four conversations forked: their last, part-filled pages copied in all layers
        _copy("copy_fork", 16, 64, 4, 8, 128),
        # a pool compacted: pages moved to its front in all layers
        _copy("copy_compact", 16, 768, 300, 8, 128),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["attend"] * 4 + ["append", "copy"])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    head_dim = rng.choice([64, 128])
    page = rng.choice([64, 128])
    if op == "copy":
        layers, pages = rng.randint(1, 16), _log(rng, 16, 700)
        return {k: v for k, v in _copy("", layers, pages, rng.randint(1, max(1, pages // 3)),
                                       kv_heads, head_dim, page).items() if k != "name"}
    dtype = rng.choice(["bf16", "f16"])
    seqs = _log(rng, 1, 128)
    if op == "append":
        dtype = rng.choice(["bf16", "f16", "f32"])
        q_max = 1 if rng.random() < 0.4 else _log(rng, 2, max(2, 20000 // seqs))
        kv_max = q_max + _log(rng, 1, 4000)
        q_min = max(1, q_max // rng.choice([1, 2, 5]))
        kv_min = max(q_max, kv_max // rng.choice([1, 3]))
        case = _append("", seqs, (kv_min, kv_max), (q_min, q_max), kv_heads, head_dim, page, dtype)
        return {k: v for k, v in case.items() if k != "name"}
    group = rng.choice([1, 2, 3, 4, 5, 7, 8, 16])
    form = rng.choice(["one", "few", "prompt"])
    if form == "prompt":
        seqs = min(seqs, 8)
        kv_max = _log(rng, 16, 6000)
        # rows x keys of the padded scores within the largest listed case
        q_max = max(1, min(kv_max, 32 * 8191 * 8191 // (seqs * kv_heads * group * kv_max)))
        q_max = _log(rng, min(9, q_max), q_max)
    else:
        kv_max = _log(rng, 9, max(9, min(131072, 524288 // seqs)))
        q_max = 1 if form == "one" else rng.randint(2, 8)
    q_min = max(1, q_max // rng.choice([1, 1, 3]))
    kv_min = max(q_max, kv_max // rng.choice([1, 2, 8]))
    window = rng.choice([0, 0, 0, _log(rng, 16, 4096)])
    sinks = rng.choice([0, 4, rng.randint(1, 200)]) if window else 0
    case = _attend("", seqs, (kv_min, max(kv_min, kv_max)), (q_min, q_max), kv_heads * group,
                   kv_heads, head_dim, page, dtype, window, sinks)
    return {k: v for k, v in case.items() if k != "name"}


def _lengths(case):
    """(keys, new tokens) of each sequence: part of the case, the same for every seed."""
    rng = random.Random(case["seqs"] * 1000003 + case["kv_max"] * 101 + case["q_max"])
    kv = [rng.randint(case["kv_min"], case["kv_max"]) for _ in range(case["seqs"])]
    kv[0] = case["kv_max"]
    q = [rng.randint(case["q_min"], case["q_max"]) for _ in kv]
    q[0] = case["q_max"]
    return kv, [min(a, b) for a, b in zip(q, kv)]


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def _exponent(amax):
    """Smallest e with amax <= 448 * 2**e, within the range of a page's exponent."""
    m, e = torch.frexp(amax)                       # amax = m * 2**e, m in [0.5, 1)
    e = torch.where(m > 0.875, e - 8, e - 9)
    return torch.where(amax > 0, e, torch.full_like(e, E_MIN)).clamp(E_MIN, E_MAX)


def _filled(gen, shape, spread):
    """Pages of normal values: channels of unlike size, as keys and values
    have them, and pages of unlike size."""
    pages, _, heads, slots, dim = shape
    codes = torch.empty(shape, dtype=torch.uint8, device="cuda")
    exps = torch.empty(shape[:3], dtype=torch.int8, device="cuda")
    chan = torch.exp2(torch.randn((1, 2, heads, 1, dim), generator=gen, device="cuda") * 0.7)
    step = max(1, (1 << 26) // (2 * heads * slots * dim))
    for at in range(0, pages, step):
        n = min(step, pages - at)
        x = torch.randn((n, 2, heads, slots, dim), generator=gen, device="cuda") * chan
        x *= torch.exp2(spread * (torch.rand((n, 2, heads, 1, 1), generator=gen, device="cuda") - 0.5))
        e = _exponent(x.abs().amax((3, 4)))
        codes[at:at + n] = (x * torch.exp2(-e.float())[..., None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
        exps[at:at + n] = e
    return codes, exps


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = np.random.default_rng(seed)
    H, D, P = case["kv_heads"], case["head_dim"], case["page"]
    s = {"case": case}
    if case["op"] == "copy":
        n = case["pages"]
        codes, exps = _filled(gen, (case["layers"] * n, 2, H, P, D), 2.0)
        s["codes"], s["exps"] = codes.view(case["layers"], n, 2, H, P, D), exps.view(case["layers"], n, 2, H)
        order = host.permutation(n)
        k = min(case["pairs"], n // 2)
        s["src"], s["dst"] = order[:k].tolist(), order[k:2 * k].tolist()
    else:
        kv, q = _lengths(case)
        width = max(-(-n // P) for n in kv)
        used = sum(-(-n // P) for n in kv)
        order = iter(host.permutation(used + 3).tolist())
        table = np.zeros((len(kv), width), np.int32)
        for b, n in enumerate(kv):
            for i in range(-(-n // P)):
                table[b, i] = next(order)
        s["codes"], s["exps"] = _filled(gen, (used + 3, 2, H, P, D), 2.0)
        starts = np.concatenate([[0], np.cumsum(q)])
        tokens = int(starts[-1])
        dtype = TYPES[case["dtype"]]
        s.update(kv=kv, q=q, table=torch.from_numpy(table).long().cuda(),
                 kv_len=torch.tensor(kv, device="cuda"), q_len=torch.tensor(q, device="cuda"),
                 starts=torch.tensor(starts[:-1], device="cuda"))
        s["of"] = torch.repeat_interleave(torch.arange(len(kv), device="cuda"), s["q_len"])
        s["nth"] = torch.arange(tokens, device="cuda") - s["starts"][s["of"]]
        if case["op"] == "attend":
            s["query"] = torch.randn((tokens, case["heads"], D), generator=gen, device="cuda").to(dtype)
            s["scale"] = D ** -0.5
            s["out"] = torch.empty_like(s["query"])
        else:
            both = torch.randn((2, tokens, H, D), generator=gen, device="cuda")
            both *= torch.exp2(torch.randn((2, 1, H, D), generator=gen, device="cuda") * 0.7)
            s["k"], s["v"] = both[0].to(dtype), both[1].to(dtype)
            s["at"] = s["kv_len"][s["of"]] - s["q_len"][s["of"]] + s["nth"]    # position of each new token
            # the pages that get new tokens, one row each, and each token's row
            first, last = [(n - m) // P for n, m in zip(kv, q)], [(n - 1) // P for n in kv]
            rows = np.concatenate([[0], np.cumsum([b - a + 1 for a, b in zip(first, last)])])
            s["row"] = torch.tensor(rows[:-1], device="cuda")[s["of"]] + s["at"] // P - torch.tensor(first, device="cuda")[s["of"]]
            pages = [table[b, i] for b in range(len(kv)) for i in range(first[b], last[b] + 1)]
            old = [max(0, (kv[b] - q[b]) - i * P) for b in range(len(kv)) for i in range(first[b], last[b] + 1)]
            s["touched"] = torch.tensor(np.array(pages), device="cuda").long()
            s["old"] = torch.tensor(old, device="cuda")                        # tokens there before
    if own:
        if "ptxgen" not in sys.modules:
            sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "emmy-ptx_b200"))
        from ptxgen import KVCache
        lay = s["codes"] if case["op"] == "copy" else s["codes"][None]
        ex = s["exps"] if case["op"] == "copy" else s["exps"][None]
        s["stream"] = torch.cuda.current_stream().cuda_stream
        s["cache"] = KVCache(lay.shape[1], H, D, page_size=P, layers=lay.shape[0], storage=(lay, ex))
        if case["op"] != "copy":
            s["batch"] = s["cache"].batch(table, kv, q, stream=s["stream"])
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------


def run(s):
    op = s["case"]["op"]
    if own:
        if op == "attend":
            return s["batch"].attend(0, s["query"], s["out"], scale=s["scale"], window=s["case"]["window"],
                                     sinks=s["case"]["sinks"], stream=s["stream"])
        if op == "append":
            s["batch"].append(0, s["k"], s["v"], stream=s["stream"])
        else:
            s["cache"].copy_pages(s["src"], s["dst"], stream=s["stream"])
        return {"codes": s["codes"].view(torch.float8_e4m3fn), "exps": s["exps"]}
    return {"attend": _plain_attend, "append": _plain_append, "copy": _plain_copy}[op](s)


def _plain_copy(s):
    src = torch.tensor(s["src"], device="cuda")
    dst = torch.tensor(s["dst"], device="cuda")
    s["codes"][:, dst] = s["codes"][:, src]
    s["exps"][:, dst] = s["exps"][:, src]
    return {"codes": s["codes"].view(torch.float8_e4m3fn), "exps": s["exps"]}


def _plain_append(s):
    P = s["case"]["page"]
    page, old = s["touched"], s["old"]
    x = torch.stack([s["k"], s["v"]], 1).float()                                # [token, side, head, d]
    n, H, D = len(page), x.shape[2], x.shape[3]
    new = torch.zeros((n, P, 2, H, D), device="cuda")
    slot = s["at"] % P
    new[s["row"], slot] = x
    e_old = s["exps"][page].int()
    e = _exponent(new.abs().amax((1, 4)))
    e = torch.where((old > 0)[:, None, None], torch.maximum(e, e_old), e)
    held = s["codes"][page].view(torch.float8_e4m3fn).float() * torch.exp2(e_old.float())[..., None, None]
    is_new = torch.zeros((n, P), dtype=torch.bool, device="cuda")
    is_new[s["row"], slot] = True
    at = torch.arange(P, device="cuda")[None]
    value = torch.where(is_new[:, None, None, :, None], new.permute(0, 2, 3, 1, 4), held)
    codes = (value * torch.exp2(-e.float())[..., None, None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    keep = ~(is_new | (at < old[:, None]))                                      # slots behind the sequence
    s["codes"][page] = torch.where(keep[:, None, None, :, None], s["codes"][page], codes)
    s["exps"][page] = e.to(torch.int8)
    return {"codes": s["codes"].view(torch.float8_e4m3fn), "exps": s["exps"]}


def _plain_attend(s):
    c = s["case"]
    B, H, D, P = c["seqs"], c["kv_heads"], c["head_dim"], c["page"]
    G, nq = c["heads"] // H, c["q_max"]
    table = s["table"]
    L = table.shape[1] * P
    held = s["codes"][table].view(torch.float8_e4m3fn).float()                  # [B, page, side, H, P, D]
    held *= torch.exp2(s["exps"][table].float())[..., None, None]
    held = held.permute(2, 0, 3, 1, 4, 5).reshape(2, B, H, L, D)
    query = torch.zeros((B, nq, H, G, D), device="cuda")
    query[s["of"], s["nth"]] = s["query"].float().view(-1, H, G, D)
    query = query.permute(0, 2, 1, 3, 4).reshape(B, H, nq * G, D)
    score = (query @ held[0].transpose(-1, -2)).mul_(s["scale"]).view(B, H, nq, G, L)
    pos = (s["kv_len"] - s["q_len"])[:, None] + torch.arange(nq, device="cuda")  # [B, nq]
    key = torch.arange(L, device="cuda")
    seen = (key <= pos[..., None]) & (key < s["kv_len"][:, None, None])
    if c["window"]:
        seen &= (pos[..., None] - key < c["window"]) | (key < c["sinks"])
    score.masked_fill_(~seen[:, None, :, None], float("-inf"))
    top = score.amax(-1, keepdim=True).clamp(min=-1e30)
    score.sub_(top).exp_()
    total = score.sum(-1)
    got = (score.view(B, H, nq * G, L) @ held[1]).view(B, H, nq, G, D)
    got = torch.where(total[..., None] > 0, got / total[..., None], 0.0)
    got = got.permute(0, 2, 1, 3, 4).reshape(B, nq, H * G, D)
    return got[s["of"], s["nth"]].to(s["query"].dtype)


# ---------------------------------------------------------------------------
# what a pass cannot do without, and what it returns in 64 bits
# ---------------------------------------------------------------------------


def _seen_keys(n, q, window, sinks):
    """(keys that some query sees, (query, key) pairs) of one sequence."""
    if not window:
        return n, q * (n - q) + q * (q + 1) // 2
    pos = np.arange(n - q, n, dtype=np.int64)
    low = np.maximum(pos - window + 1, 0)
    near = pos - low + 1
    first = np.minimum(np.minimum(sinks, pos + 1), low)
    return int(n - low[0] + min(sinks, low[0])), int((near + first).sum())


def work(case):
    H, D, P = case["kv_heads"], case["head_dim"], case["page"]
    if case["op"] == "copy":
        pairs = min(case["pairs"], case["pages"] // 2)
        return {"bytes": 2 * pairs * case["layers"] * (2 * H * P * D + 2 * H), "flops": 0}
    kv, q = _lengths(case)
    tokens = sum(q)
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "append":
        pages = sum((n - 1) // P - (n - m) // P + 1 for n, m in zip(kv, q))
        return {"bytes": 2 * H * (tokens * D * (size + 1) + 2 * pages), "flops": 0}
    seen = [_seen_keys(n, m, case["window"], case["sinks"]) for n, m in zip(kv, q)]
    keys, pairs = sum(a for a, _ in seen), sum(b for _, b in seen)
    return {"bytes": 2 * H * keys * D + 2 * H * (keys // P) + 2 * tokens * case["heads"] * D * size,
            "flops": 4 * D * case["heads"] * pairs}


def exact(case, seed):
    s = prepare(case, seed)
    H, D, P = case["kv_heads"], case["head_dim"], case["page"]
    codes = s["codes"].view(torch.float8_e4m3fn)
    if case["op"] == "copy":
        codes, exps = codes.double(), s["exps"]
        for a, b in zip(s["src"], s["dst"]):
            codes[:, b].copy_(codes[:, a])
            exps[:, b].copy_(exps[:, a])
        return {"codes": codes, "exps": exps}
    table = s["table"].tolist()
    starts = s["starts"].tolist()
    if case["op"] == "append":
        codes, exps = codes.double(), s["exps"]
        for b, (n, m) in enumerate(zip(s["kv"], s["q"])):
            for side, x in enumerate((s["k"], s["v"])):
                x = x[starts[b]:starts[b] + m].double().transpose(0, 1)         # [H, m, D]
                for i in range((n - m) // P, (n - 1) // P + 1):
                    lo, hi = max(n - m, i * P), min(n, (i + 1) * P)
                    part = x[:, lo - (n - m):hi - (n - m)]
                    at, old = codes[table[b][i], side], lo - i * P
                    before = exps[table[b][i], side].double()
                    amax = part.abs().amax((1, 2))
                    e = torch.floor(torch.log2(amax / 448)).clamp(E_MIN, E_MAX) - 1
                    for _ in range(3):                                          # the logarithm may be a hair off
                        e = torch.where(torch.exp2(e) * 448 < amax, e + 1, e)
                    e = e.clamp(E_MIN, E_MAX)
                    if old:
                        e = torch.maximum(e, before)
                        at[:, :old] *= torch.exp2(before - e)[:, None, None]
                    at[:, old:old + hi - lo] = part * torch.exp2(-e)[:, None, None]
                    exps[table[b][i], side] = e.to(torch.int8)
        return {"codes": codes, "exps": exps}
    G = case["heads"] // H
    out = torch.zeros(s["query"].shape, dtype=torch.float64, device="cuda")
    for b, (n, m) in enumerate(zip(s["kv"], s["q"])):
        at = torch.tensor(table[b][:-(-n // P)], device="cuda")
        pos = torch.arange(n - m, n, device="cuda")[:, None]
        key = torch.arange(n, device="cuda")[None]
        hidden = key > pos
        if case["window"]:
            hidden |= (key >= case["sinks"]) & (key <= pos - case["window"])
        for h in range(H):
            k, v = [(codes[at, side, h].double() * torch.exp2(s["exps"][at, side, h].double())[:, None, None]).reshape(-1, D)[:n]
                    for side in (0, 1)]
            for g in range(G):
                q = s["query"][starts[b]:starts[b] + m, h * G + g].double()
                p = torch.softmax((q @ k.T * s["scale"]).masked_fill_(hidden, float("-inf")), -1)
                out[starts[b]:starts[b] + m, h * G + g] = p @ v
    return out
