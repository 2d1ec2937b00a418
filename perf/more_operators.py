"""Workloads of rotary positions and of what they are for: rotated appends to
the paged 8-bit key/value cache, and attention of sequences that share a
prefix of its pages.

A rotary position turns the pairs (a, b) of a head's first ``dims`` values by
the angle position * frequency[i].  A cache layer is a pool of pages
``codes[page, K or V, kv head, slot, d]`` in e4m3 with one power-of-two scale
``2 ** exps[page, K or V, kv head]`` for each page, side and head.  Each case
below is one call of one operator; ``run`` computes it in elementary torch
operations, or with ``own`` set by the framework's kernels.
"""

import math
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


def _rotary(dims, interleaved=False, base=10000.0, scaling="none", factor=1.0, length=0):
    return {"dims": dims, "interleaved": interleaved, "base": base, "scaling": scaling,
            "factor": factor, "length": length}


def _rotate(name, tokens, heads, head_dim, rotary, far, dtype="bf16", backward=False, packed=False, scattered=False):
    return {"name": name, "op": "rotate", "tokens": tokens, "heads": heads, "head_dim": head_dim, "far": far,
            "dtype": dtype, "backward": backward, "packed": packed, "scattered": scattered, **rotary}


def _append(name, seqs, kv, q, heads, kv_heads, head_dim, rotary, page=64, dtype="bf16"):
    return {"name": name, "op": "append", "seqs": seqs, "kv_min": kv[0], "kv_max": kv[1],
            "q_min": q[0], "q_max": q[1], "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "page": page, "dtype": dtype, **rotary}


def _shared(name, runs, members, alone, prefix, owned, q, heads, kv_heads, head_dim, page=64, dtype="bf16"):
    return {"name": name, "op": "shared", "runs": runs, "members": members, "alone": alone, "prefix": prefix,
            "own_min": owned[0], "own_max": owned[1], "q_min": q[0], "q_max": q[1], "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "dtype": dtype}


def listed():
    return [
        # the queries of one conversation's next token: latency
        _rotate("rotate_one", 1, 32, 128, _rotary(128), 8191, scattered=True),
        # the queries of a long prompt, a slice of the array that holds keys and values too,
        # in a context longer than the trained one
        _rotate("rotate_prompt", 8191, 32, 128, _rotary(128, base=500000.0, scaling="bands", factor=8.0, length=8192),
                131072, packed=True),
        # part of each head, neighbours paired, in 32 bits
        _rotate("rotate_part", 4093, 20, 80, _rotary(32, interleaved=True), 4096, dtype="f32"),
        # gradients of a training batch of long sequences
        _rotate("rotate_gradients", 32768, 16, 128, _rotary(128, scaling="ramp", factor=16.0, length=4096),
                65536, backward=True),
        # one conversation's next token into the cache, its queries rotated on the way: latency
        _append("append_one", 1, (1025, 1025), (1, 1), 32, 8, 128, _rotary(128)),
        # a full server: one new token for each of 64 conversations
        _append("append_step", 64, (700, 8191), (1, 1), 32, 8, 128, _rotary(128, base=500000.0)),
        # several prompts at once
        _append("append_prompts", 6, (6000, 9000), (3000, 8000), 32, 8, 128, _rotary(128, base=500000.0)),
        # prompts behind histories, half of each head rotated, neighbours paired, f16
        _append("append_part", 5, (1500, 4000), (200, 1500), 20, 5, 64, _rotary(32, interleaved=True),
                page=128, dtype="f16"),
        # four answers to one question
        _shared("shared_few", 1, 4, 0, 2048, (40, 400), (1, 1), 32, 8, 128),
        # a full server whose conversations begin with the same instructions
        _shared("shared_batch", 1, 64, 0, 8192, (1, 1000), (1, 1), 32, 8, 128),
        # draft tokens of conversations about three documents, and of some about none
        _shared("shared_drafts", 3, 10, 3, 4096, (30, 700), (4, 4), 20, 5, 64, page=128, dtype="f16"),
        # many questions about one very long document, few kv heads
        _shared("shared_long", 1, 128, 0, 32768, (20, 2000), (1, 1), 16, 2, 128, page=128, dtype="f16"),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def _draw_rotary(rng, head_dim):
    dims = head_dim if rng.random() < 0.5 else 2 * rng.randint(1, head_dim // 2)
    scaling = rng.choice(["none", "none", "linear", "base", "bands", "ramp"])
    if scaling == "base" and dims == 2:
        scaling = "linear"
    return _rotary(dims, rng.random() < 0.4, rng.choice([10000.0, 500000.0, 1e6]), scaling,
                   1.0 if scaling == "none" else rng.choice([2.0, 4.0, 8.0, 16.0]),
                   0 if scaling in ("none", "linear", "base") else rng.choice([2048, 4096, 8192]))


def draw(rng):
    op = rng.choice(["rotate", "append", "shared", "shared"])
    if op == "rotate":
        head_dim = rng.choice([64, 80, 96, 128, 128, 256])
        heads = _log(rng, 1, 64)
        tokens = _log(rng, 1, 32768 * 16 * 128 // (heads * head_dim))
        case = _rotate("", tokens, heads, head_dim, _draw_rotary(rng, head_dim), _log(rng, tokens + 1, 1 << 20),
                       rng.choice(["bf16", "f16", "f32"]), rng.random() < 0.4, rng.random() < 0.3,
                       rng.random() < 0.3)
        if case["dtype"] == "f32":
            case["tokens"] = max(1, tokens // 2)
    elif op == "append":
        kv_heads, head_dim, page = rng.choice([1, 2, 3, 4, 8]), rng.choice([64, 128]), rng.choice([64, 128])
        group = rng.choice([1, 2, 4, 5, 8])
        seqs = _log(rng, 1, 128)
        dtype = rng.choice(["bf16", "f16", "f32"])
        most = 20000 * 8 * 4 // (seqs * kv_heads * group * (2 if dtype == "f32" else 1))
        q_max = 1 if rng.random() < 0.4 else _log(rng, 2, max(2, min(20000 // seqs, most)))
        kv_max = q_max + _log(rng, 1, 4000)
        q_min = max(1, q_max // rng.choice([1, 2, 5]))
        kv_min = max(q_max, kv_max // rng.choice([1, 3]))
        case = _append("", seqs, (kv_min, kv_max), (q_min, q_max), kv_heads * group, kv_heads, head_dim,
                       _draw_rotary(rng, head_dim), page, dtype)
    else:
        kv_heads, head_dim, page = rng.choice([1, 2, 3, 4, 8]), rng.choice([64, 128]), rng.choice([64, 128])
        group = rng.choice([1, 2, 3, 4, 5, 7, 8, 16])
        runs = rng.choice([1, 1, 1, 2, 3])
        members = _log(rng, 2, 128 // runs)
        alone = rng.choice([0, 0, rng.randint(1, 5)])
        q_max = 1 if rng.random() < 0.6 else rng.randint(1, max(1, 32 // group))
        seqs, rows = runs * members + alone, kv_heads * group * q_max
        # rows x keys, keys of all sequences and bytes within the largest listed case
        keys = 80000000 // (2 * kv_heads * head_dim)
        own_max = _log(rng, q_max, max(q_max, min(2000, keys // (2 * seqs))))
        most = min(128 * 16 * 34768 // (seqs * rows) - own_max, 128 * 2 * 34768 // (seqs * kv_heads) - own_max,
                   (keys - seqs * own_max) // (runs + alone))
        prefix = page * _log(rng, 1, max(1, min(32768, most) // page))
        case = _shared("", runs, members, alone, prefix, (max(q_max, own_max // rng.choice([1, 2, 20])), own_max),
                       (max(1, q_max // rng.choice([1, 1, 2])), q_max), kv_heads * group, kv_heads, head_dim,
                       page, rng.choice(["bf16", "f16"]))
    return {k: v for k, v in case.items() if k != "name"}


def _lengths(case):
    """(keys, new tokens, shared keys) of each sequence, runs first: part of
    the case, the same for every seed."""
    if case["op"] == "append":
        rng = random.Random(case["seqs"] * 1000003 + case["kv_max"] * 101 + case["q_max"])
        kv = [rng.randint(case["kv_min"], case["kv_max"]) for _ in range(case["seqs"])]
        kv[0] = case["kv_max"]
        q = [rng.randint(case["q_min"], case["q_max"]) for _ in kv]
        q[0] = case["q_max"]
        return kv, [min(a, b) for a, b in zip(q, kv)], [0] * len(kv)
    together = case["runs"] * case["members"]
    seqs = together + case["alone"]
    rng = random.Random(seqs * 1000003 + case["prefix"] * 101 + case["own_max"])
    kept = [rng.randint(case["own_min"], case["own_max"]) for _ in range(seqs)]
    kept[0] = case["own_max"]
    q = [min(n, rng.randint(case["q_min"], case["q_max"])) for n in kept]
    q[0] = case["q_max"]
    shared = [case["prefix"]] * together + [0] * case["alone"]
    # those that share nothing are as long as the others
    return [n + case["prefix"] for n in kept], q, shared


def _frequencies(case):
    """f_i of the pairs, and the gain, in 64 bits."""
    r, base, s, L = case["dims"], case["base"], case["factor"], case["length"]
    if case["scaling"] == "base":
        base *= s ** (r / (r - 2))
    i = np.arange(r // 2, dtype=np.float64)
    f = base ** (-2 * i / r)
    if case["scaling"] == "linear":
        return f / s, 1.0
    if case["scaling"] == "bands":
        # turns over the trained length: above 4 as they are, below 1 slowed, between mixed
        turns = L * f / (2 * math.pi)
        mix = np.clip((turns - 1.0) / 3.0, 0, 1)
        return (1 - mix) * f / s + mix * f, 1.0
    if case["scaling"] == "ramp":
        # by the pair's index, between those of 32 turns and of one
        def at(turns):
            return r * math.log(L / (2 * math.pi * turns)) / (2 * math.log(base))
        low, high = max(0, math.floor(at(32))), min(r - 1, math.ceil(at(1)))
        ramp = np.clip((i - low) / max(high - low, 1e-3), 0, 1)
        return f * (1 - ramp) + f / s * ramp, 0.1 * math.log(s) + 1
    return f, 1.0


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


def _package():
    if "ptxgen" not in sys.modules:
        sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "emmy-ptx_b200"))
    import ptxgen
    return ptxgen


def _own_rotary(case):
    scaling = {"type": case["scaling"], "factor": case["factor"]}
    if case["scaling"] in ("bands", "ramp"):
        scaling["length"] = case["length"]
    return _package().Rotary(case["head_dim"], dims=case["dims"], base=case["base"], interleaved=case["interleaved"],
                             scaling=None if case["scaling"] == "none" else scaling)


def _prepare_rotate(case, gen, host, s):
    T, H, D, dtype = case["tokens"], case["heads"], case["head_dim"], TYPES[case["dtype"]]
    if case["scattered"]:
        pos = host.integers(0, case["far"], T)
    else:
        pos = int(host.integers(0, max(1, case["far"] - T))) + np.arange(T)
    s["pos"] = torch.from_numpy(pos.astype(np.int64)).cuda()
    # queries beside keys and values of two heads, or by themselves
    wide = torch.randn((T, H + 4 if case["packed"] else H, D), generator=gen, device="cuda").to(dtype)
    s["x"] = wide[:, :H]
    s["out"] = torch.empty((T, H, D), dtype=dtype, device="cuda")
    if own:
        s["rotary"], s["stream"] = _own_rotary(case), torch.cuda.current_stream().cuda_stream


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = np.random.default_rng(seed)
    s = {"case": case}
    if case["op"] != "shared":
        f, s["gain"] = _frequencies(case)
        s["freq"] = torch.from_numpy(f).cuda()
    if case["op"] == "rotate":
        _prepare_rotate(case, gen, host, s)
        return s
    H, D, P = case["kv_heads"], case["head_dim"], case["page"]
    kv, q, shared = _lengths(case)
    B, width = len(kv), max(-(-n // P) for n in kv)
    prefixes = case["runs"] if case["op"] == "shared" else 0
    used = sum(-(-(n - m) // P) for n, m in zip(kv, shared)) + prefixes * case.get("prefix", 0) // P
    order = iter(host.permutation(used + 3).tolist())
    table = np.zeros((B, width), np.int32)
    for b, n in enumerate(kv):
        held = shared[b] // P
        if held and b % case["members"]:
            table[b, :held] = table[b - 1, :held]
            first = held
        else:
            first = 0
        for i in range(first, -(-n // P)):
            table[b, i] = next(order)
    s["codes"], s["exps"] = _filled(gen, (used + 3, 2, H, P, D), 2.0)
    starts = np.concatenate([[0], np.cumsum(q)])
    tokens, dtype = int(starts[-1]), TYPES[case["dtype"]]
    s.update(kv=kv, q=q, shared=shared, table=torch.from_numpy(table).long().cuda(),
             kv_len=torch.tensor(kv, device="cuda"), q_len=torch.tensor(q, device="cuda"),
             starts=torch.tensor(starts[:-1], device="cuda"))
    s["of"] = torch.repeat_interleave(torch.arange(B, device="cuda"), s["q_len"])
    s["nth"] = torch.arange(tokens, device="cuda") - s["starts"][s["of"]]
    s["at"] = s["kv_len"][s["of"]] - s["q_len"][s["of"]] + s["nth"]        # position of each new token
    s["query"] = torch.randn((tokens, case["heads"], D), generator=gen, device="cuda").to(dtype)
    s["out"] = torch.empty_like(s["query"])
    if case["op"] == "append":
        both = torch.randn((2, tokens, H, D), generator=gen, device="cuda")
        both *= torch.exp2(torch.randn((2, 1, H, D), generator=gen, device="cuda") * 0.7)
        s["k"], s["v"] = both[0].to(dtype), both[1].to(dtype)
        # the pages that get new tokens, one row each, and each token's row
        first, last = [(n - m) // P for n, m in zip(kv, q)], [(n - 1) // P for n in kv]
        rows = np.concatenate([[0], np.cumsum([b - a + 1 for a, b in zip(first, last)])])
        s["row"] = torch.tensor(rows[:-1], device="cuda")[s["of"]] + s["at"] // P - torch.tensor(first, device="cuda")[s["of"]]
        pages = [table[b, i] for b in range(B) for i in range(first[b], last[b] + 1)]
        old = [max(0, (kv[b] - q[b]) - i * P) for b in range(B) for i in range(first[b], last[b] + 1)]
        s["touched"] = torch.tensor(np.array(pages), device="cuda").long()
        s["old"] = torch.tensor(old, device="cuda")                        # tokens there before
    else:
        s["scale"] = D ** -0.5
    if own:
        s["stream"] = torch.cuda.current_stream().cuda_stream
        s["cache"] = _package().KVCache(s["codes"].shape[0], H, D, page_size=P,
                                        storage=(s["codes"][None], s["exps"][None]))
        if case["op"] == "append":
            s["rotary"] = _own_rotary(case)
            s["batch"] = s["cache"].batch(table, kv, q, stream=s["stream"])
        else:
            s["batch"] = s["cache"].batch(table, kv, q, stream=s["stream"], shared=True)
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------


def run(s):
    op = s["case"]["op"]
    if own:
        if op == "rotate":
            turn = s["rotary"].backward if s["case"]["backward"] else s["rotary"].rotate
            return turn(s["x"], s["pos"], s["out"], stream=s["stream"])
        if op == "shared":
            return s["batch"].attend(0, s["query"], s["out"], scale=s["scale"], stream=s["stream"])
        s["batch"].append(0, s["k"], s["v"], rotary=s["rotary"], q=s["query"], q_out=s["out"], stream=s["stream"])
        return {"codes": s["codes"].view(torch.float8_e4m3fn), "exps": s["exps"], "q": s["out"]}
    return {"rotate": _plain_rotate, "append": _plain_append, "shared": _plain_attend}[op](s)


def _turned(s, x, pos, sign=1.0):
    """x [tokens, heads, head_dim], f32 or f64, turned to positions pos: angles
    and their functions in 64 bits."""
    c = s["case"]
    r = c["dims"]
    angle = pos.double()[:, None, None] * s["freq"]
    cos, sin = (s["gain"] * torch.cos(angle)).to(x.dtype), (sign * s["gain"] * torch.sin(angle)).to(x.dtype)
    out = x.clone()
    if c["interleaved"]:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        out[..., 0:r:2] = a * cos - b * sin
        out[..., 1:r:2] = a * sin + b * cos
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        out[..., :r // 2] = a * cos - b * sin
        out[..., r // 2:r] = a * sin + b * cos
    return out


def _plain_rotate(s):
    return _turned(s, s["x"].float(), s["pos"], -1.0 if s["case"]["backward"] else 1.0).to(s["x"].dtype)


def _plain_append(s):
    P = s["case"]["page"]
    page, old = s["touched"], s["old"]
    # (64 bits: a page's exponent changes at a border)
    x = torch.stack([_turned(s, s["k"].double(), s["at"]).float(), s["v"].float()], 1)   # [token, side, head, d]
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
    q = _turned(s, s["query"].float(), s["at"]).to(s["query"].dtype)
    return {"codes": s["codes"].view(torch.float8_e4m3fn), "exps": s["exps"], "q": q}


def _plain_attend(s):
    c = s["case"]
    B, H, D, P = len(s["kv"]), c["kv_heads"], c["head_dim"], c["page"]
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


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "rotate":
        values = case["tokens"] * case["heads"]
        return {"bytes": 2 * values * case["head_dim"] * size + 8 * case["tokens"], "flops": 3 * values * case["dims"]}
    H, D, P = case["kv_heads"], case["head_dim"], case["page"]
    kv, q, shared = _lengths(case)
    tokens = sum(q)
    if case["op"] == "append":
        pages = sum((n - 1) // P - (n - m) // P + 1 for n, m in zip(kv, q))
        return {"bytes": 2 * H * (tokens * D * (size + 1) + 2 * pages) + 2 * tokens * case["heads"] * D * size,
                "flops": 3 * tokens * (H + case["heads"]) * case["dims"]}
    keys = sum(n - m for n, m in zip(kv, shared)) + case["runs"] * case["prefix"]
    pairs = sum(m * (n - m) + m * (m + 1) // 2 for n, m in zip(kv, q))
    return {"bytes": 2 * H * keys * D + 2 * H * (keys // P) + 2 * tokens * case["heads"] * D * size,
            "flops": 4 * D * case["heads"] * pairs}


def _exact_turned(s, x, pos, conjugate=False):
    """Each pair as a complex number times gain * e^(i position frequency)."""
    c = s["case"]
    r, x = c["dims"], x.double()
    turn = torch.polar(torch.full((), s["gain"], dtype=torch.float64, device="cuda"), pos.double()[:, None, None] * s["freq"])
    if conjugate:
        turn = turn.conj()
    if c["interleaved"]:
        z = torch.view_as_complex(x[..., :r].reshape(*x.shape[:-1], r // 2, 2).contiguous()) * turn
        turned = torch.view_as_real(z).reshape(*x.shape[:-1], r)
    else:
        z = torch.complex(x[..., :r // 2].contiguous(), x[..., r // 2:r].contiguous()) * turn
        turned = torch.cat([z.real, z.imag], -1)
    return torch.cat([turned, x[..., r:]], -1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotate":
        return _exact_turned(s, s["x"], s["pos"], case["backward"])
    H, D, P = case["kv_heads"], case["head_dim"], case["page"]
    codes = s["codes"].view(torch.float8_e4m3fn)
    table = s["table"].tolist()
    starts = s["starts"].tolist()
    if case["op"] == "append":
        codes, exps = codes.double(), s["exps"]
        sides = _exact_turned(s, s["k"], s["at"]), s["v"].double()
        for b, (n, m) in enumerate(zip(s["kv"], s["q"])):
            for side, x in enumerate(sides):
                x = x[starts[b]:starts[b] + m].transpose(0, 1)                  # [H, m, D]
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
        return {"codes": codes, "exps": exps, "q": _exact_turned(s, s["query"], s["at"])}
    G = case["heads"] // H
    out = torch.zeros(s["query"].shape, dtype=torch.float64, device="cuda")
    for b, (n, m) in enumerate(zip(s["kv"], s["q"])):
        at = torch.tensor(table[b][:-(-n // P)], device="cuda")
        hidden = torch.arange(n, device="cuda")[None] > torch.arange(n - m, n, device="cuda")[:, None]
        for h in range(H):
            k, v = [(codes[at, side, h].double() * torch.exp2(s["exps"][at, side, h].double())[:, None, None]).reshape(-1, D)[:n]
                    for side in (0, 1)]
            q = s["query"][starts[b]:starts[b] + m, h * G:(h + 1) * G].double()
            p = torch.softmax((torch.einsum("mgd,nd->gmn", q, k) * s["scale"]).masked_fill_(hidden, float("-inf")), -1)
            out[starts[b]:starts[b] + m, h * G:(h + 1) * G] = torch.einsum("gmn,nd->mgd", p, v)
    return out
