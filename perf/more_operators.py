"""What a batch's captured step needs around its layers, as measurable cases, with plain forms: rotations from positions,
attention over a prompt that all sequences share, and rules on the logits with the greedy token.

``factors``  cos and sin of rotary positions with several axes (time, height, width, ..) for each row, head and pair
             (``Rotary.factors``).
``turn``     the paged row step that rotates by such positions (``KvPages.qkv_rows`` with ``Rotary.at``): QKV rows split,
             normalized, rotated and appended in 8 bits, and the rows of the touched blocks read back.
``shared``   attention of 1..8 query rows for each of a batch of sequences whose first positions are one sequence's pages
             (``KvPages.attention_shared``).
``choose``   penalties for repeated tokens, biases and grammar masks on logits, and the greedy token
             (``select_tokens`` with ``LogitRules``).

Shapes are the checkpoint's (16 query and 8 KV heads of 64, a 65,536-row vocabulary, a page of 6,544 positions) or generic
ones. Keys are held once for each KV head (``keys`` 8) or, where an image makes the query heads of a KV head rotate
differently, for each query head (``keys`` 16).

With ``own`` false ``run`` is made of elementary torch operations; with it true it makes the framework's calls.
"""
import math
import random
import sys
from pathlib import Path

import numpy as np
import torch

own = False

HEADS, KV_HEADS, HEAD, PAIRS, BLOCK = 16, 8, 64, 32, 16
EPS32 = 2.0 ** -23
INF = float("inf")

_loaded = None


def _package():
    global _loaded
    if _loaded is None:
        path = str(Path(__file__).resolve().parents[1] / "falcon-ocr-cpu_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        import focr_hip

        _loaded = focr_hip
    return _loaded


def listed():
    return [
        # One session's next position: the smallest call.
        {"name": "factors_1", "op": "factors", "rows": 1, "axes": 3},
        # A journal page's prompt, an image with its text.
        {"name": "factors_6544", "op": "factors", "rows": 6544, "axes": 3},
        # One token of each of 64 sessions, text positions only.
        {"name": "turn_step_64", "op": "turn", "seqs": 64, "rows": 1, "length": 4000, "page": 64, "keys": 8, "axes": 1},
        # Whole prompts with images enter the cache.
        {"name": "turn_prompt_4", "op": "turn", "seqs": 4, "rows": 6544, "length": 40, "page": 64, "keys": 16, "axes": 3},
        # Two sessions behind a short instruction, on small pages.
        {"name": "shared_2_at_240", "op": "shared", "seqs": 2, "rows": 1, "prefix": 240, "own": 37, "page": 16, "keys": 8},
        # Eight sessions verify up to four drafts each on one page of a journal.
        {"name": "shared_8x5_at_6528", "op": "shared", "seqs": 8, "rows": 5, "prefix": 6528, "own": 500, "page": 64, "keys": 16},
        # A full batch of questions on that page.
        {"name": "shared_64_at_6528", "op": "shared", "seqs": 64, "rows": 1, "prefix": 6528, "own": 300, "page": 64, "keys": 16},
        # Many sessions behind a long document.
        {"name": "shared_200_at_32768", "op": "shared", "seqs": 200, "rows": 1, "prefix": 32768, "own": 900, "page": 128, "keys": 8},
        # A greedy token of one session.
        {"name": "choose_1", "op": "choose", "rows": 1, "vocab": 65536, "history": 300, "recent": 0, "bias": 0, "masked": False, "adjusted": False},
        # An odd vocabulary, a few rows, their logits kept for sampling.
        {"name": "choose_odd_7", "op": "choose", "rows": 7, "vocab": 50021, "history": 2000, "recent": 512, "bias": 40, "masked": True, "adjusted": True},
        # A full batch with long answers under a grammar.
        {"name": "choose_64", "op": "choose", "rows": 64, "vocab": 65536, "history": 8192, "recent": 0, "bias": 200, "masked": True, "adjusted": False},
        # Every rule, a large vocabulary and the largest batch, for sampling.
        {"name": "choose_256", "op": "choose", "rows": 256, "vocab": 131072, "history": 4096, "recent": 1024, "bias": 300, "masked": True, "adjusted": True},
    ]


def _log_int(rng, low, high):
    """An integer spread over the logarithm of [low, high]."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["factors", "turn", "shared", "shared", "choose", "choose"])
    if op == "factors":
        return {"op": op, "rows": _log_int(rng, 1, 26176), "axes": rng.randint(1, 4)}
    if op == "choose":
        rows = _log_int(rng, 1, 256)
        vocab = _log_int(rng, 1000, min(262144, 256 * 131072 // rows))
        if rng.random() < 0.5:
            vocab = max(1024, vocab // 64 * 64)
        history = _log_int(rng, 1, 16384)
        return {"op": op, "rows": rows, "vocab": vocab, "history": history, "recent": rng.choice([0, 0, 64, 777]),
                "bias": rng.choice([0, rng.randint(1, 400)]), "masked": rng.random() < 0.6, "adjusted": rng.random() < 0.5}
    keys, page = rng.choice([8, 16]), rng.choice([16, 32, 64, 128])
    seqs = _log_int(rng, 1, 200)
    if op == "turn":
        rows = 1 if rng.random() < 0.5 else _log_int(rng, 2, max(2, 12000 // seqs))
        return {"op": op, "seqs": seqs, "rows": rows, "length": _log_int(rng, 1, 8000), "page": page, "keys": keys,
                "axes": rng.randint(1, 4)}
    rows = rng.choice([1, 1, 2, 3, 5, 8])
    # Held once for each KV head the keys are half as many: the products are what bounds the largest case.
    prefix = _log_int(rng, 64, min(65536, 200 * 32768 // (seqs * rows)))
    return {"op": op, "seqs": seqs, "rows": rows, "prefix": max(page, prefix // page * page),
            "own": _log_int(rng, 1, min(4000, 180000 // seqs)), "page": page, "keys": keys}


def _spans(case):
    """(positions cached, new rows) of each sequence: the longest as the case says, the others less (``shared``: behind
    the prefix)."""
    low = 0.25 if case["op"] == "turn" else 0.0
    length = case["length"] if case["op"] == "turn" else case["own"]
    rng = random.Random(case["seqs"] * 1000003 + length)
    spans = []
    for i in range(case["seqs"]):
        share = 1.0 if i == 0 else rng.uniform(low, 1.0)
        rows = case["rows"] if i == 0 else max(1, int(case["rows"] * rng.uniform(0.25, 1.0)))
        spans.append((int(length * share), rows))
    return spans


def _histories(case):
    """How many tokens each row has before: the longest as the case says, the second none."""
    rng = random.Random(case["rows"] * 1000003 + case["history"])
    return [case["history"] if i == 0 else 0 if i == 1 else int(case["history"] * rng.random()) for i in range(case["rows"])]


def work(case):
    op = case["op"]
    if op == "factors":
        rows, table = case["rows"], case["axes"] * HEADS * PAIRS
        # An angle and its two functions are some 30 products and sums.
        return {"bytes": 4 * rows * case["axes"] + 4 * table + 8 * rows * HEADS * PAIRS, "flops": 60 * rows * HEADS * PAIRS}
    if op == "choose":
        rows, vocab = case["rows"], case["vocab"]
        tokens = sum(min(n, case["recent"]) if case["recent"] else n for n in _histories(case))
        read = 4 * rows * vocab + 4 * tokens + 12 * rows + 8 * rows * case["bias"] + (rows * vocab / 8 if case["masked"] else 0)
        return {"bytes": read + 4 * rows + (4 * rows * vocab if case["adjusted"] else 0), "flops": rows * vocab + 6 * tokens}
    spans, keys = _spans(case), case["keys"]
    rows = sum(n for _, n in spans)
    if op == "turn":
        opened = sum(length % BLOCK for length, _ in spans)
        heads = (HEADS + 2 * KV_HEADS) * HEAD
        stored = (keys + KV_HEADS) * HEAD
        # QKV rows, positions and queries; the open blocks' earlier rows; codes; the rows read back.
        return {"bytes": 4 * rows * (heads + case["axes"] + HEADS * HEAD) + 4 * opened * stored + (rows + opened) * stored * 5,
                "flops": rows * (10 * heads + 60 * HEADS * PAIRS)}
    code = (keys + KV_HEADS) * (HEAD + 4 / BLOCK)
    total = case["prefix"] + sum(length + n for length, n in spans)
    return {"bytes": total * code + 8 * rows * HEADS * HEAD,
            "flops": sum(4 * HEAD * HEADS * n * (case["prefix"] + length + n) for length, n in spans)}


# -- inputs -------------------------------------------------------------------
class _Maker:
    """Seeded values, made on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(int(seed) & 0x7FFFFFFF)

    def normal(self, *shape, std=1.0):
        return torch.randn(shape, generator=self.g, device="cuda") * std

    def uniform(self, low, high, *shape):
        return torch.rand(shape, generator=self.g, device="cuda") * (high - low) + low

    def perm(self, n):
        return torch.randperm(n, generator=self.g, device="cuda")


def _starts(counts):
    """int32 [0, c0, c0 + c1, ...] on the GPU."""
    return torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device="cuda")


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _owners(starts, rows):
    """The sequence of each row, and the row's number in it."""
    at = torch.arange(rows, device="cuda")
    seq = torch.searchsorted(starts[1:].long(), at, right=True)
    return seq, at - starts.long()[seq]


def _unit_heads(make, *shape):
    """Heads as an RMS norm leaves them."""
    x = make.normal(*shape, HEAD)
    return x / x.square().mean(-1, keepdim=True).sqrt()


def _frequencies(make, axes):
    """[axes][HEADS][32]: the first axis (time) turns every pair of one-axis positions, or the first half of them; the
    others (places in an image) turn the rest, in a direction of each head and pair."""
    table = torch.zeros(axes, HEADS, PAIRS, device="cuda")
    timed = PAIRS if axes == 1 else PAIRS // 2
    table[0, :, :timed] = 10000.0 ** (-torch.arange(timed, device="cuda") / timed)
    if axes > 1:
        way = make.normal(axes - 1, HEADS, PAIRS - timed)
        size = 30.0 * 100.0 ** (-torch.arange(PAIRS - timed, device="cuda") / (PAIRS - timed))
        table[1:, :, timed:] = way / way.square().sum(0).sqrt() * size
    return table


def _positions(make, times, axes):
    """[rows][axes]: whole steps of time and, for most rows, a place from -1 to 1 on the other axes."""
    out = torch.zeros(times.numel(), axes, device="cuda")
    out[:, 0] = times.float()
    if axes > 1:
        out[:, 1:] = make.uniform(-1.0, 1.0, times.numel(), axes - 1)
        out[times % 8 == 0, 1:] = 0.0
    return out


def _factors_inputs(case, make):
    start = int(make.uniform(0, 100000, 1).item())
    times = torch.arange(start, start + case["rows"], device="cuda")
    return _frequencies(make, case["axes"]), _positions(make, times, case["axes"])


def _prepare_factors(case, make):
    frequencies, positions = _factors_inputs(case, make)
    state = {"case": case, "positions": positions}
    if own:
        state["rotary"] = _package().Rotary(frequencies)
        state["out"] = torch.empty(case["rows"], HEADS, PAIRS, 2, device="cuda")
        return state
    state["frequencies"] = frequencies
    return state


def _turn_inputs(case, make):
    spans, keys, axes = _spans(case), case["keys"], case["axes"]
    rows, open_rows = sum(n for _, n in spans), sum(length % BLOCK for length, _ in spans)
    times = torch.cat([torch.arange(length, length + n, device="cuda") for length, n in spans])
    return {"qkv": make.normal(rows, (HEADS + 2 * KV_HEADS) * HEAD), "frequencies": _frequencies(make, axes),
            "positions": _positions(make, times, axes),
            # The rows that the first touched blocks hold already.
            "open_k": _unit_heads(make, open_rows, keys), "open_v": make.normal(open_rows, KV_HEADS, HEAD)}


def _prepare_turn(case, make):
    spans, page = _spans(case), case["page"]
    rows, opened = sum(n for _, n in spans), [length % BLOCK for length, _ in spans]
    open_rows = sum(opened)
    given = _turn_inputs(case, make)
    state = {"case": case, "lens": _int32([length for length, _ in spans]), "starts": _starts([n for _, n in spans]),
             "qkv": given["qkv"], "positions": given["positions"],
             # The rows of the touched blocks, which are read back.
             "block_lens": _int32([length // BLOCK * BLOCK for length, _ in spans]),
             "block_starts": _starts([length % BLOCK + n for length, n in spans]), "block_rows": rows + open_rows}
    counts = [-(-(length + n) // page) for length, n in spans]
    ids = make.perm(sum(counts) + 3)
    if own:
        fh = _package()
        kv = fh.KvPages(sum(counts) + 3, page, len(spans), max(counts), HEADS, KV_HEADS, key_heads=case["keys"])
        held, at = ids.tolist(), 0
        for seq, count in enumerate(counts):
            kv.map(seq, 0, held[at:at + count])
            at += count
        if open_rows:
            kv.append(given["open_k"], given["open_v"], state["block_lens"], row_start=_starts(opened))
        state["kv"], state["rotary"] = kv, fh.Rotary(given["frequencies"])
        return state
    state |= {"frequencies": given["frequencies"], "open_k": given["open_k"], "open_v": given["open_v"]}
    state["open_seq"], state["open_at"] = _owners(_starts(opened), open_rows)
    state["units"] = sum((length + n - 1) // BLOCK - length // BLOCK + 1 for length, n in spans)
    return state


def _shared_inputs(case, make):
    spans, keys = _spans(case), case["keys"]
    rows, held = sum(n for _, n in spans), sum(length + n for length, n in spans)
    return {"q": _unit_heads(make, rows, HEADS), "sinks": make.normal(HEADS),
            "prefix_k": _unit_heads(make, case["prefix"], keys), "prefix_v": make.normal(case["prefix"], KV_HEADS, HEAD),
            "own_k": _unit_heads(make, held, keys), "own_v": make.normal(held, KV_HEADS, HEAD)}


def _prepare_shared(case, make):
    spans, page, prefix, seqs = _spans(case), case["page"], case["prefix"], case["seqs"]
    totals = [length + n for length, n in spans]
    given = _shared_inputs(case, make)
    state = {"case": case, "lens": _int32([prefix + length for length, _ in spans]), "starts": _starts([n for _, n in spans]),
             "q": given["q"], "sinks": given["sinks"], "longest": prefix + max(totals)}
    front, counts = prefix // page, [-(-t // page) for t in totals]
    pages = front + sum(counts)
    ids = make.perm(pages)
    first = np.concatenate([[0], np.cumsum(counts)]) + front
    if own:
        kv = _package().KvPages(pages, page, seqs, front + max(counts), HEADS, KV_HEADS, key_heads=case["keys"])
        held = ids.tolist()
        for seq, count in enumerate(counts):
            kv.map(seq, 0, held[:front] + held[int(first[seq]):int(first[seq]) + count])
        kv.append(given["prefix_k"], given["prefix_v"], _int32([0]), row_start=_int32([0, prefix]))
        kv.append(given["own_k"], given["own_v"], torch.full_like(state["lens"], prefix), row_start=_starts(totals))
        state["kv"] = kv
        return state
    # The same cache for the plain form: codes [page][head][position][64], scales [page][head][block].
    table = torch.zeros(seqs, max(counts), dtype=torch.int64, device="cuda")
    for seq, count in enumerate(counts):
        table[seq, :count] = ids[int(first[seq]):int(first[seq]) + count]
    state["front"], state["table"] = ids[:front], table
    seq, pos = _owners(_starts(totals), sum(totals))
    place = table[seq, pos // page] * page + pos % page
    at = torch.arange(prefix, device="cuda")
    front_place = ids[at // page] * page + at % page
    for name, heads in (("k", case["keys"]), ("v", KV_HEADS)):
        full = torch.zeros(pages * page, heads, HEAD, device="cuda")
        full[front_place] = given["prefix_" + name]
        full[place] = given["own_" + name]
        codes, scales = _coded(full.view(pages * page // BLOCK, BLOCK, heads, HEAD))
        state[name + "_codes"] = codes.view(pages, page, heads, HEAD).transpose(1, 2).contiguous()
        state[name + "_scales"] = scales.view(pages, page // BLOCK, heads).transpose(1, 2).contiguous()
        del full, codes, scales
    return state


def _choose_inputs(case, make):
    rows, vocab, n_bias = case["rows"], case["vocab"], case["bias"]
    given = {"logits": make.normal(rows, vocab, std=3.0)}
    # Some tokens come often, as in text, and what came before is likely again.
    history = (vocab * make.uniform(0.0, 1.0, rows, case["history"]) ** 6).long().clamp(max=vocab - 1)
    given["history"] = history.int()
    given["lengths"] = _int32(_histories(case))
    given["logits"].scatter_(1, history[:, :64], make.uniform(8.0, 14.0, rows, min(64, case["history"])))
    # Repetition, presence and frequency; every fourth row has none.
    penalties = torch.stack([make.uniform(1.0, 1.6, rows), make.uniform(0.0, 1.5, rows), make.uniform(0.0, 0.3, rows)], dim=1)
    penalties[3::4] = torch.tensor([1.0, 0.0, 0.0], device="cuda")
    given["penalties"] = penalties.contiguous()
    if n_bias:
        # Different tokens of a row: a random stretch of them, spread out.
        step = vocab // n_bias
        at = make.uniform(0.0, 1.0, rows, n_bias).mul(step).long().clamp(max=step - 1)
        given["bias_tokens"] = (torch.arange(n_bias, device="cuda") * step + at).int().contiguous()
        given["bias"] = make.normal(rows, n_bias, std=4.0)
    if case["masked"]:
        # From a grammar that allows one token in 512 to one that forbids a few; the last of several rows allows none.
        share = 0.5 ** make.uniform(0.0, 9.0, rows, 1)
        if rows > 4:
            share[rows - 1] = 0.0
        words = -(-vocab // 32)
        bits = (make.uniform(0.0, 1.0, rows, words * 32) < share).view(rows, words, 32)
        packed = (bits.long() << torch.arange(32, device="cuda")).sum(-1)
        given["allowed"] = torch.where(packed >= 2 ** 31, packed - 2 ** 32, packed).int().contiguous()
    return given


def _prepare_choose(case, make):
    given = _choose_inputs(case, make)
    state = {"case": case, "logits": given["logits"]}
    if own:
        state["rules"] = _package().LogitRules(
            history=given["history"], lengths=given["lengths"], recent=case["recent"], penalties=given["penalties"],
            bias_tokens=given.get("bias_tokens"), bias=given.get("bias"), allowed=given.get("allowed"))
        state["tokens"] = torch.empty(case["rows"], dtype=torch.int32, device="cuda")
        state["adjusted"] = torch.empty_like(given["logits"]) if case["adjusted"] else None
        return state
    return state | given


def prepare(case, seed):
    make = _Maker(seed)
    return {"factors": _prepare_factors, "turn": _prepare_turn, "shared": _prepare_shared,
            "choose": _prepare_choose}[case["op"]](case, make)


# -- one pass -----------------------------------------------------------------
def run(state):
    return {"factors": _run_factors, "turn": _run_turn, "shared": _run_shared, "choose": _run_choose}[state["case"]["op"]](state)


def _angles(positions, frequencies):
    """[rows][HEADS][32] in 64 bits: where positions are far, 32 bits have no fraction of a turn left. One axis after the
    other, so that the sum's order is what the operator says."""
    p, f = positions.double(), frequencies.double()
    angle = p[:, 0, None, None] * f[0]
    for axis in range(1, p.shape[1]):
        angle = angle + p[:, axis, None, None] * f[axis]
    return angle


def _cos_sin(positions, frequencies):
    angle = _angles(positions, frequencies)
    return torch.stack([angle.cos(), angle.sin()], dim=-1).float()


def _run_factors(state):
    if own:
        return {"factors": state["rotary"].factors(state["positions"], out=state["out"])}
    return {"factors": _cos_sin(state["positions"], state["frequencies"])}


def _norm_rotate(x, factors):
    """Heads [.., 64] RMS-normalized (the squares added pairwise: two halves of 32, each folded 16-8-4-2-1) and rotated by
    [.., 32, 2] cos and sin; every product and sum rounds to FP32, as the row step defines it."""
    s = (x * x).view(*x.shape[:-1], 2, 32)
    s = s[..., :16] + s[..., 16:]
    s = s[..., :8] + s[..., 8:]
    s = s[..., :4] + s[..., 4:]
    s = s[..., :2] + s[..., 2:]
    s = s[..., 0] + s[..., 1]
    total = s[..., 0] + s[..., 1]
    root = torch.sqrt(total / 64.0 + EPS32)
    y = x * torch.div(torch.ones_like(root), root).unsqueeze(-1)
    a, b, cos, sin = y[..., 0::2], y[..., 1::2], factors[..., 0], factors[..., 1]
    return torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).view(x.shape)


def _coded(x):
    """Blocks [.., 16, heads, 64] in 8 bits: codes and the scale of each block and head."""
    peak = x.abs().amax(dim=(-3, -1))
    scales = torch.div(peak, torch.full_like(peak, 127.0))
    inverse = torch.where(scales >= 2.0 ** -126, torch.div(torch.ones_like(scales), scales), torch.zeros_like(scales))
    codes = (x * inverse[..., None, :, None]).round().to(torch.int8)
    return codes, scales


def _run_turn(state):
    case, qkv, lens = state["case"], state["qkv"], state["lens"]
    if own:
        kv = state["kv"]
        q = kv.qkv_rows(qkv, state["rotary"].at(state["positions"]), lens, row_start=state["starts"])
        k, v = kv.dequantize(state["block_rows"], state["block_lens"], row_start=state["block_starts"])
        return {"q": q, "k": k, "v": v}
    rows, keys = qkv.shape[0], case["keys"]
    factors = _cos_sin(state["positions"], state["frequencies"])
    heads = qkv.view(rows, HEADS + 2 * KV_HEADS, HEAD)
    q = _norm_rotate(heads[:, :HEADS], factors)
    key, value = heads[:, HEADS:HEADS + KV_HEADS], heads[:, HEADS + KV_HEADS:]
    repeat = HEADS // KV_HEADS
    if keys == HEADS:
        key = _norm_rotate(key.repeat_interleave(repeat, dim=1), factors)
    else:
        key = _norm_rotate(key, factors[:, ::repeat])
    # The touched blocks: the rows that the first one of a sequence holds, then the new ones.
    lens, starts = lens.long(), state["starts"].long()
    seq, number = _owners(starts, rows)
    pos = lens[seq] + number
    blocks = (lens + starts[1:] - starts[:-1] - 1) // BLOCK - lens // BLOCK + 1
    base = blocks.cumsum(0) - blocks
    read_seq, read_at = _owners(state["block_starts"], state["block_rows"])
    read_unit, read_at = base[read_seq] + read_at // BLOCK, read_at % BLOCK
    k, v = _through(state, key, "open_k", base, seq, pos, lens), _through(state, value, "open_v", base, seq, pos, lens)
    return {"q": q, "k": k[read_unit, read_at], "v": v[read_unit, read_at]}


def _through(state, new, name, base, seq, pos, lens):
    """What the touched blocks hold of their earlier rows and the new ones, as the codes say it."""
    full = torch.zeros(state["units"], BLOCK, new.shape[1], HEAD, device="cuda")
    full[base[state["open_seq"]], state["open_at"]] = state[name]
    full[base[seq] + pos // BLOCK - lens[seq] // BLOCK, pos % BLOCK] = new
    codes, scales = _coded(full)
    return codes.float() * scales[:, None, :, None]


def _run_shared(state):
    case, q, lens, starts = state["case"], state["q"], state["lens"], state["starts"]
    if own:
        return {"out": state["kv"].attention_shared(q, lens, state["longest"], case["prefix"], row_start=starts,
                                                    sinks=state["sinks"])}
    rows, keys, page, seqs, most = q.shape[0], case["keys"], case["page"], case["seqs"], case["rows"]
    group, table = HEADS // keys, state["table"]
    length = table.shape[1] * page

    def decoded(name, pages):
        """[.., pages] to [.., heads, positions, 64]."""
        codes = state[name + "_codes"][pages].float()
        values = codes.unflatten(-2, (page // BLOCK, BLOCK)) * state[name + "_scales"][pages][..., None, None]
        return values.flatten(-3, -2).transpose(-4, -3).flatten(-3, -2)

    # The prefix, for all rows at once: columns [key head][64][row, query head of it].
    columns = q.view(rows, keys, group, HEAD).permute(1, 3, 0, 2).reshape(keys, HEAD, rows * group)
    front = (decoded("k", state["front"]) @ columns).view(keys, case["prefix"], rows, group) * 0.125
    # Each sequence's own positions, for its rows, padded to the most of a sequence.
    seq, number = _owners(starts, rows)
    padded = torch.zeros(seqs, most, HEADS, HEAD, device="cuda")
    padded[seq, number] = q
    columns = padded.view(seqs, most, keys, group, HEAD).permute(0, 2, 4, 3, 1).reshape(seqs, keys, HEAD, group * most)
    back = (decoded("k", table) @ columns).view(seqs, keys, length, group, most) * 0.125
    visible = lens.long()[:, None] - case["prefix"] + torch.arange(1, most + 1, device="cuda")
    hidden = torch.arange(length, device="cuda")[None, :, None] >= visible[:, None, :]
    back = back.masked_fill(hidden[:, None, :, None, :], -INF)
    # [row][head] of both.
    front_peak = front.amax(dim=1).permute(1, 0, 2).reshape(rows, HEADS)
    back_peak = back.amax(dim=2).permute(0, 3, 1, 2).reshape(seqs, most, HEADS)[seq, number]
    peak = torch.maximum(front_peak, back_peak)
    front = (front - peak.view(rows, keys, group).transpose(0, 1)[:, None]).exp()
    filled = torch.zeros(seqs, most, HEADS, device="cuda")
    filled[seq, number] = peak
    back = (back - filled.view(seqs, most, keys, group).permute(0, 2, 3, 1)[:, :, None]).exp()
    total = front.sum(dim=1).permute(1, 0, 2).reshape(rows, HEADS)
    total = total + back.sum(dim=2).permute(0, 3, 1, 2).reshape(seqs, most, HEADS)[seq, number]
    # Weights [KV head][its query heads x rows][position] times the values.
    each = HEADS // KV_HEADS
    front = front.permute(0, 3, 2, 1).reshape(KV_HEADS, each * rows, case["prefix"]) @ decoded("v", state["front"])
    back = back.permute(0, 1, 3, 4, 2).reshape(seqs, KV_HEADS, each * most, length) @ decoded("v", table)
    out = front.view(HEADS, rows, HEAD).transpose(0, 1) + back.view(seqs, HEADS, most, HEAD).transpose(1, 2)[seq, number]
    sink = 1.0 / (1.0 + (state["sinks"] - (peak + total.log())).exp())
    return {"out": out / total[..., None] * sink[..., None]}


def _run_choose(state):
    case, z = state["case"], state["logits"]
    rows, vocab = case["rows"], case["vocab"]
    if own:
        tokens = _package().select_tokens(z, rows, vocab, state["rules"], adjusted=state["adjusted"], tokens=state["tokens"])
        return {"tokens": tokens} if state["adjusted"] is None else {"tokens": tokens, "adjusted": state["adjusted"]}
    lengths, history = state["lengths"].long()[:, None], state["history"].long()
    at = torch.arange(history.shape[1], device="cuda")
    counted = at < lengths
    if case["recent"]:
        counted = counted & (at >= lengths - case["recent"])
    # Whole numbers, so their sums do not depend on the order.
    counts = torch.zeros(rows, vocab, device="cuda").scatter_add_(1, history, counted.float())
    repetition, presence, frequency = (state["penalties"][:, i:i + 1] for i in range(3))
    seen = counts > 0
    z = torch.where(seen, torch.where(z > 0, z / repetition, z * repetition), z)
    z = torch.where(seen, z - (counts * frequency + presence), z)
    if case["bias"]:
        z = z.scatter(1, state["bias_tokens"].long(), z.gather(1, state["bias_tokens"].long()) + state["bias"])
    if case["masked"]:
        bits = (state["allowed"][:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
        z = torch.where(bits.view(rows, -1)[:, :vocab] > 0, z, torch.full_like(z, -INF))
    peak = z.amax(dim=1, keepdim=True)
    first = torch.where(z == peak, torch.arange(vocab, device="cuda"), vocab).amin(dim=1)
    tokens = torch.where(peak[:, 0] == -INF, -1, first).int()
    return {"tokens": tokens, "adjusted": z} if case["adjusted"] else {"tokens": tokens}


# -- the definitions, in 64 bits --------------------------------------------------
def _f32(x):
    """A 64-bit value rounded to FP32, as the row step and the codes are defined."""
    return x.float().double()


def _exact_factors(case, make):
    frequencies, positions = _factors_inputs(case, make)
    f = frequencies.double()
    angle = (positions.double() @ f.view(case["axes"], -1)).view(-1, HEADS, PAIRS)
    out = torch.empty(*angle.shape, 2, dtype=torch.float64, device="cuda")
    out[..., 0], out[..., 1] = torch.cos(angle), torch.sin(angle)
    return {"factors": out}


def _exact_rotate(x, factors):
    squares = _f32(x * x)
    halves = []
    for part in (squares[..., :32], squares[..., 32:]):
        while part.shape[-1] > 1:
            wide = part.shape[-1] // 2
            part = _f32(part[..., :wide] + part[..., wide:])
        halves.append(part[..., 0])
    scale = _f32(1.0 / _f32(torch.sqrt(_f32(_f32(_f32(halves[0] + halves[1]) / 64) + EPS32))))
    y = _f32(x * scale[..., None])
    out = torch.empty_like(x)
    cos, sin = factors[..., 0], factors[..., 1]
    out[..., 0::2] = _f32(_f32(y[..., 0::2] * cos) - _f32(y[..., 1::2] * sin))
    out[..., 1::2] = _f32(_f32(y[..., 0::2] * sin) + _f32(y[..., 1::2] * cos))
    return out


def _exact_blocks(x):
    """What blocks of rows [..][16][heads][64] hold."""
    scale = _f32(x.abs().amax(dim=(-3, -1), keepdim=True) / 127)
    inverse = torch.where(scale > 0, _f32(1.0 / scale), torch.zeros_like(scale))
    return _f32(torch.round(_f32(x * inverse)) * scale)


def _exact_turn(case, make):
    spans, keys = _spans(case), case["keys"]
    rows, open_rows = sum(n for _, n in spans), sum(length % BLOCK for length, _ in spans)
    if rows > 20000 or rows + open_rows > 16 * 2500:
        return None
    given = {name: x.double() for name, x in _turn_inputs(case, make).items()}
    qkv = given["qkv"].view(rows, -1, HEAD)
    f = given["frequencies"]
    angle = (given["positions"] @ f.view(case["axes"], -1)).view(rows, HEADS, PAIRS)
    rope = _f32(torch.stack([torch.cos(angle), torch.sin(angle)], dim=-1))
    source = torch.arange(keys, device="cuda") * KV_HEADS // keys
    turn = torch.arange(keys, device="cuda") * (HEADS // keys)
    q = _exact_rotate(qkv[:, :HEADS], rope)
    key, value = _exact_rotate(qkv[:, HEADS + source], rope[:, turn]), qkv[:, HEADS + KV_HEADS:]
    k, v, at, open_at = [], [], 0, 0
    for length, n in spans:
        held = length % BLOCK
        for result, earlier, new in ((k, given["open_k"], key), (v, given["open_v"], value)):
            whole = torch.cat([earlier[open_at:open_at + held], new[at:at + n]])
            pad = torch.zeros(-(held + n) % BLOCK, *whole.shape[1:], dtype=torch.float64, device="cuda")
            blocks = torch.cat([whole, pad]).view(-1, BLOCK, *whole.shape[1:])
            result.append(_exact_blocks(blocks).flatten(0, 1)[:held + n])
        at, open_at = at + n, open_at + held
    return {"q": q, "k": torch.cat(k), "v": torch.cat(v)}


def _exact_shared(case, make):
    spans = _spans(case)
    given = {name: x.double() for name, x in _shared_inputs(case, make).items()}
    q, sinks = given["q"], given["sinks"]

    def held(x):
        """[positions][heads][64] as the cache has it, for every query head: [HEADS][positions][64]."""
        pad = torch.zeros(-x.shape[0] % BLOCK, *x.shape[1:], dtype=torch.float64, device="cuda")
        x = _exact_blocks(torch.cat([x, pad]).view(-1, BLOCK, *x.shape[1:])).flatten(0, 1)[:x.shape[0]]
        return x.repeat_interleave(HEADS // x.shape[1], dim=1).transpose(0, 1).contiguous()

    # The prefix: log of the sum of weights, and the mean value, of every head and row.
    key, value = held(given["prefix_k"]), held(given["prefix_v"])
    front_lse, front_mean = [], []
    for h in range(HEADS):
        s = q[:, h] @ key[h].t() / 8.0
        lse = torch.logsumexp(s, dim=1)
        front_lse.append(lse)
        front_mean.append(torch.exp(s - lse[:, None]) @ value[h])
    front_lse, front_mean = torch.stack(front_lse, dim=1), torch.stack(front_mean, dim=1)
    out, first, row = [], 0, 0
    for length, n in spans:
        total = length + n
        key, value = held(given["own_k"][first:first + total]), held(given["own_v"][first:first + total])
        for r in range(n):
            seen = length + r + 1
            s = (key[:, :seen] @ q[row + r][:, :, None])[..., 0] / 8.0
            lse = torch.logaddexp(front_lse[row + r], torch.logsumexp(s, dim=1))
            mean = (torch.exp(s - lse[:, None])[:, None, :] @ value[:, :seen])[:, 0]
            mean = mean + torch.exp(front_lse[row + r] - lse)[:, None] * front_mean[row + r]
            out.append(mean * torch.sigmoid(lse - sinks)[:, None])
        first, row = first + total, row + n
    return {"out": torch.stack(out)}


def _exact_choose(case, make):
    if not case["adjusted"]:
        return None  # a token is a whole number
    given = _choose_inputs(case, make)
    rows, vocab = case["rows"], case["vocab"]
    out = given["logits"].double()
    for r, length in enumerate(_histories(case)):
        begin = max(0, length - case["recent"]) if case["recent"] else 0
        counts = torch.bincount(given["history"][r, begin:length].long(), minlength=vocab).double()
        repetition, presence, frequency = (float(x) for x in given["penalties"][r].double())
        row = torch.where(out[r] > 0, out[r] / repetition, out[r] * repetition) - counts * frequency - presence
        out[r] = torch.where(counts > 0, row, out[r])
        if case["bias"]:
            out[r][given["bias_tokens"][r].long()] += given["bias"][r].double()
        if case["masked"]:
            words = given["allowed"][r].long()
            at = torch.arange(vocab, device="cuda")
            out[r][((words[at // 32] >> (at % 32)) & 1) == 0] = -INF
    return {"tokens": None, "adjusted": out}


def exact(case, seed):
    make = _Maker(seed)
    return {"factors": _exact_factors, "turn": _exact_turn, "shared": _exact_shared, "choose": _exact_choose}[case["op"]](case, make)
