"""Operators for serving several sessions at once, as measurable cases, with their plain forms.

``linear4``  a projection of 1..8 rows with 4-bit weights and a scale per group of input columns
             (``QuantLinear`` with ``bits=4``), the norm before it and the GLU or the residual after it folded in.
``pages``    a step's QKV rows split, normalized, rotated and appended to a cache of pages that holds keys and values in
             8 bits with a scale for each block of 16 positions and head (``KvPages.qkv_rows``), and the rows of the
             touched blocks read back (``KvPages.dequantize``).
``attend``   attention of 1..8 query rows for each of a batch of sequences over that cache (``KvPages.attention``).

Shapes are the checkpoint's (dim 768, 16 query and 8 KV heads of 64, FFN 2,304, a 65,536-row vocabulary head, a page of 6,544
positions) or generic ones. Keys are held once for each KV head (``keys`` 8) or, where an image makes the query heads of
a KV head rotate differently, for each query head (``keys`` 16).

With ``own`` false ``run`` is made of elementary torch operations; with it true it makes the framework's calls.
"""
import math
import random
import sys
from pathlib import Path

import numpy as np
import torch

own = False

HEAD, BLOCK = 64, 16


def _package():
    path = str(Path(__file__).resolve().parents[1] / "falcon-ocr-cpu_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import focr_hip

    return focr_hip


def listed():
    return [
        # The smallest call: one session's QKV projection.
        {"name": "linear4_qkv_1", "op": "linear4", "out": 2048, "in": 768, "group": 64, "rows": 1, "epilogue": "STORE", "norm": True},
        # Five sessions' FFN output with its residual.
        {"name": "linear4_w2_5", "op": "linear4", "out": 768, "in": 2304, "group": 64, "rows": 5, "epilogue": "ADD", "norm": False},
        # The vocabulary head of a greedy step.
        {"name": "linear4_head_1", "op": "linear4", "out": 65536, "in": 768, "group": 128, "rows": 1, "epilogue": "STORE", "norm": True},
        # Sizes that fill neither tiles nor groups.
        {"name": "linear4_odd_3", "op": "linear4", "out": 5003, "in": 1111, "group": 32, "rows": 3, "epilogue": "STORE", "norm": False},
        # A large layer's gated FFN input for a full batch of rows.
        {"name": "linear4_ffn_8", "op": "linear4", "out": 24576, "in": 8192, "group": 64, "rows": 8, "epilogue": "GLU", "norm": True},
        # One token of each of 64 sessions.
        {"name": "pages_step_64", "op": "pages", "seqs": 64, "rows": 1, "length": 4000, "page": 64, "keys": 8},
        # Whole prompts with images enter the cache: the longest a page of 6,544 positions.
        {"name": "pages_prompt_4", "op": "pages", "seqs": 4, "rows": 6544, "length": 40, "page": 64, "keys": 16},
        # The smallest attention: one session behind a short prompt.
        {"name": "attend_1_at_100", "op": "attend", "seqs": 1, "rows": 1, "length": 100, "page": 64, "keys": 8},
        # Eight sessions verify up to four drafts each behind journal pages.
        {"name": "attend_8x5_at_6544", "op": "attend", "seqs": 8, "rows": 5, "length": 6544, "page": 64, "keys": 16},
        # Many short sessions on small pages.
        {"name": "attend_200_at_700", "op": "attend", "seqs": 200, "rows": 1, "length": 700, "page": 16, "keys": 8},
        # A full batch of long sessions.
        {"name": "attend_64_at_8192", "op": "attend", "seqs": 64, "rows": 1, "length": 8192, "page": 64, "keys": 16},
        # One very long session.
        {"name": "attend_1_at_131072", "op": "attend", "seqs": 1, "rows": 2, "length": 131072, "page": 128, "keys": 8},
    ]


def _log_int(rng, low, high):
    """An integer spread over the logarithm of [low, high]."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["linear4", "linear4", "pages", "attend", "attend"])
    if op == "linear4":
        epilogue = rng.choice(["STORE", "GLU", "ADD"])
        out, inner = _log_int(rng, 256, 65536), _log_int(rng, 96, 8192)
        if rng.random() < 0.5:  # real matrices mostly have whole tiles
            out, inner = max(256, out // 128 * 128), max(128, inner // 128 * 128)
        if epilogue == "GLU":
            out = out // 2 * 2
        while out * inner > 24576 * 8192:
            out = out // 4 * 2
        return {"op": op, "out": out, "in": inner, "group": rng.choice([32, 64, 64, 128]), "rows": rng.randint(1, 8),
                "epilogue": epilogue, "norm": rng.random() < 0.5}
    keys, page = rng.choice([8, 16]), rng.choice([16, 32, 64, 128])
    if op == "pages":
        seqs = _log_int(rng, 1, 200)
        rows = 1 if rng.random() < 0.5 else _log_int(rng, 2, max(2, 12000 // seqs))
        return {"op": op, "seqs": seqs, "rows": rows, "length": _log_int(rng, 1, 8000), "page": page, "keys": keys}
    seqs = _log_int(rng, 1, 200)
    return {"op": op, "seqs": seqs, "rows": rng.choice([1, 1, 2, 3, 5, 8]),
            "length": _log_int(rng, 16, min(131072, 300000 // seqs)), "page": page, "keys": keys}


HEADS, KV_HEADS = 16, 8


def _spans(case):
    """(positions cached, new rows) of each sequence: the longest as the case says, the others down to a quarter of it."""
    rng = random.Random(case["seqs"] * 1000003 + case["length"])
    spans = []
    for i in range(case["seqs"]):
        share = 1.0 if i == 0 else rng.uniform(0.25, 1.0)
        rows = case["rows"] if i == 0 else max(1, int(case["rows"] * rng.uniform(0.25, 1.0)))
        spans.append((int(case["length"] * share), rows))
    return spans


def work(case):
    if case["op"] == "linear4":
        out, inner, rows = case["out"], case["in"], case["rows"]
        wide = out // 2 if case["epilogue"] == "GLU" else out
        written = rows * wide * (2 if case["epilogue"] == "ADD" else 1)
        scales = out * -(-inner // case["group"])
        return {"bytes": out * inner / 2 + 4 * scales + 4 * rows * inner + 4 * written, "flops": 2 * rows * out * inner}
    spans, keys = _spans(case), case["keys"]
    rows = sum(n for _, n in spans)
    if case["op"] == "pages":
        opened = sum(length % BLOCK for length, _ in spans)
        heads = (HEADS + 2 * KV_HEADS) * HEAD
        stored = (keys + KV_HEADS) * HEAD
        # QKV rows, factors and queries; the open blocks' earlier rows; codes; the rows read back.
        return {"bytes": 4 * rows * (heads + 2 * HEADS * HEAD) + 4 * opened * stored + (rows + opened) * stored * 5,
                "flops": 10 * rows * heads}
    total = sum(length + n for length, n in spans)
    code = (keys + KV_HEADS) * (HEAD + 4 / BLOCK)
    return {"bytes": total * code + 8 * rows * HEADS * HEAD,
            "flops": sum(4 * HEAD * HEADS * n * (length + n) for length, n in spans)}


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

    def codes(self, *shape):
        """4-bit codes -8..7."""
        return torch.randint(-8, 8, shape, generator=self.g, device="cuda", dtype=torch.int8)

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


def _prepare_linear4(case, make):
    out, inner, group, rows = case["out"], case["in"], case["group"], case["rows"]
    codes = make.codes(out, inner)
    scales = make.uniform(0.002, 0.008, out, -(-inner // group))
    state = {"case": case, "x": make.normal(rows, inner)}
    if case["epilogue"] == "ADD":
        state["h"] = make.normal(rows, out)
    if own:
        fh = _package()
        state["matrix"] = fh.QuantLinear.from_parts(out, inner, group, codes.cpu().numpy(), scales.cpu().numpy(), bits=4)
        return state
    # Two codes a byte, the even column in the low half.
    if inner % 2:
        codes = torch.cat([codes, torch.zeros(out, 1, dtype=torch.int8, device="cuda")], dim=1)
    nibbles = codes.view(torch.uint8) & 15
    state["packed"] = nibbles[:, 0::2] | (nibbles[:, 1::2] << 4)
    state["scales"] = scales
    return state


def _unit_heads(make, *shape):
    """Heads as an RMS norm leaves them."""
    x = make.normal(*shape, HEAD)
    return x / x.square().mean(-1, keepdim=True).sqrt()


def _factors(make, case, positions):
    """[rows][HEADS][32][2]: cos and sin of a temporal rotation of the first 16 pairs, and of the rest by angles of the
    row's place in its image, which differ between the heads (none without images)."""
    freq = 10000.0 ** (-torch.arange(16, device="cuda", dtype=torch.float64) / 16)
    time = (positions.double()[:, None] * freq).to(torch.float64)[:, None, :].expand(-1, HEADS, -1)
    if case["keys"] == HEADS:
        place = make.uniform(-40.0, 40.0, positions.numel(), HEADS, 16).double()
    else:
        place = torch.zeros(positions.numel(), HEADS, 16, dtype=torch.float64, device="cuda")
    angle = torch.cat([time, place], dim=-1)
    return torch.stack([angle.cos(), angle.sin()], dim=-1).float().contiguous()


def _map_pages(kv, spans, page, ids):
    at = 0
    for seq, (length, rows) in enumerate(spans):
        count = -(-(length + rows) // page)
        kv.map(seq, 0, ids[at:at + count])
        at += count


def _prepare_pages(case, make):
    spans, keys, page = _spans(case), case["keys"], case["page"]
    rows = sum(n for _, n in spans)
    lens, starts = _int32([length for length, _ in spans]), _starts([n for _, n in spans])
    seq, number = _owners(starts, rows)
    opened = [length % BLOCK for length, _ in spans]
    open_rows = sum(opened)
    # The rows that the first touched blocks hold already.
    open_k, open_v = _unit_heads(make, open_rows, keys), make.normal(open_rows, KV_HEADS, HEAD)
    state = {"case": case, "lens": lens, "starts": starts, "qkv": make.normal(rows, (HEADS + 2 * KV_HEADS) * HEAD),
             "rope": _factors(make, case, lens.long()[seq] + number),
             # The rows of the touched blocks, which are read back.
             "block_lens": _int32([length // BLOCK * BLOCK for length, _ in spans]),
             "block_starts": _starts([length % BLOCK + n for length, n in spans]), "block_rows": rows + open_rows}
    pages = sum(-(-(length + n) // page) for length, n in spans)
    ids = make.perm(pages + 3)[:pages]
    open_starts = _starts(opened)
    if own:
        fh = _package()
        longest = max(-(-(length + n) // page) for length, n in spans)
        kv = fh.KvPages(pages + 3, page, len(spans), longest, HEADS, KV_HEADS, key_heads=keys)
        _map_pages(kv, spans, page, ids.tolist())
        if open_rows:
            kv.append(open_k, open_v, state["block_lens"], row_start=open_starts)
        state["kv"] = kv
        return state
    state["open_seq"], state["open_at"] = _owners(open_starts, open_rows)
    state["open_k"], state["open_v"] = open_k, open_v
    state["units"] = sum((length + n - 1) // BLOCK - length // BLOCK + 1 for length, n in spans)
    return state


def _prepare_attend(case, make):
    spans, keys, page = _spans(case), case["keys"], case["page"]
    totals = [length + n for length, n in spans]
    rows = sum(n for _, n in spans)
    k, v = _unit_heads(make, sum(totals), keys), make.normal(sum(totals), KV_HEADS, HEAD)
    state = {"case": case, "lens": _int32([length for length, _ in spans]), "starts": _starts([n for _, n in spans]),
             "q": _unit_heads(make, rows, HEADS), "sinks": make.normal(HEADS), "longest": max(totals)}
    counts = [-(-t // page) for t in totals]
    pages = sum(counts)
    ids = make.perm(pages)
    if own:
        fh = _package()
        kv = fh.KvPages(pages, page, len(spans), max(counts), HEADS, KV_HEADS, key_heads=keys)
        _map_pages(kv, spans, page, ids.tolist())
        kv.append(k, v, torch.zeros_like(state["lens"]), row_start=_starts(totals))
        state["kv"] = kv
        return state
    # The same cache for the plain form: codes [page][head][position][64], scales [page][head][block].
    first = np.concatenate([[0], np.cumsum(counts)])
    table = torch.zeros(len(spans), max(counts), dtype=torch.int64, device="cuda")
    for seq, count in enumerate(counts):
        table[seq, :count] = ids[int(first[seq]):int(first[seq]) + count]
    seq, pos = _owners(_starts(totals), sum(totals))
    place = table[seq, pos // page] * page + pos % page
    state["table"] = table
    for name, x, heads in (("k", k, keys), ("v", v, KV_HEADS)):
        full = torch.zeros(pages * page, heads, HEAD, device="cuda")
        full[place] = x
        codes, scales = _coded(full.view(pages * page // BLOCK, BLOCK, heads, HEAD))
        state[name + "_codes"] = codes.view(pages, page, heads, HEAD).transpose(1, 2).contiguous()
        state[name + "_scales"] = scales.view(pages, page // BLOCK, heads).transpose(1, 2).contiguous()
        del full, codes, scales
    return state


def prepare(case, seed):
    make = _Maker(seed)
    return {"linear4": _prepare_linear4, "pages": _prepare_pages, "attend": _prepare_attend}[case["op"]](case, make)


# -- one pass -----------------------------------------------------------------
def run(state):
    return {"linear4": _run_linear4, "pages": _run_pages, "attend": _run_attend}[state["case"]["op"]](state)


EPS32 = 2.0 ** -23


def _run_linear4(state):
    case, x = state["case"], state["x"]
    if own:
        fh = _package()
        out = state["matrix"].linear_ex(x, case["rows"], epilogue=fh.Epilogue[case["epilogue"]], out=state.get("h"),
                                        rms_norm=case["norm"])
        return {"out": out}
    packed, scales, group, inner = state["packed"], state["scales"], case["group"], case["in"]
    nibbles = torch.stack([packed & 15, packed >> 4], dim=-1).view(case["out"], -1)[:, :inner]
    codes = ((nibbles ^ 8).to(torch.int8) - 8).float()
    weights = codes * scales.repeat_interleave(group, dim=1)[:, :inner]
    if case["norm"]:
        x = x * (1.0 / (x.square().mean(-1, keepdim=True) + EPS32).sqrt())
    y = x @ weights.t()
    if case["epilogue"] == "GLU":
        gate = y[:, 0::2].clamp(min=0.0)
        return {"out": gate * gate * y[:, 1::2]}
    if case["epilogue"] == "ADD":
        state["h"] += y
        return {"out": state["h"]}
    return {"out": y}


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


def _run_pages(state):
    case, qkv, rope, lens = state["case"], state["qkv"], state["rope"], state["lens"]
    if own:
        kv = state["kv"]
        q = kv.qkv_rows(qkv, rope, lens, row_start=state["starts"])
        k, v = kv.dequantize(state["block_rows"], state["block_lens"], row_start=state["block_starts"])
        return {"q": q, "k": k, "v": v}
    rows, keys = qkv.shape[0], case["keys"]
    heads = qkv.view(rows, HEADS + 2 * KV_HEADS, HEAD)
    q = _norm_rotate(heads[:, :HEADS], rope)
    key, value = heads[:, HEADS:HEADS + KV_HEADS], heads[:, HEADS + KV_HEADS:]
    repeat = HEADS // KV_HEADS
    if keys == HEADS:
        key = _norm_rotate(key.repeat_interleave(repeat, dim=1), rope)
    else:
        key = _norm_rotate(key, rope[:, ::repeat])
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


def _run_attend(state):
    case, q, lens, starts = state["case"], state["q"], state["lens"], state["starts"]
    if own:
        return {"out": state["kv"].attention(q, lens, state["longest"], row_start=starts, sinks=state["sinks"])}
    rows, keys, page, table = q.shape[0], case["keys"], case["page"], state["table"]
    seqs, most = case["seqs"], case["rows"]
    length = table.shape[1] * page

    def decoded(name, heads):
        codes = state[name + "_codes"][table].float()
        values = codes.view(seqs, -1, heads, page // BLOCK, BLOCK, HEAD) * state[name + "_scales"][table][..., None, None]
        return values.view(seqs, -1, heads, page, HEAD).transpose(1, 2).reshape(seqs, heads, length, HEAD)

    # Queries [seq][key head][64][query heads of it x rows], padded to the most rows of a sequence.
    seq, number = _owners(starts, rows)
    padded = torch.zeros(seqs, most, HEADS, HEAD, device="cuda")
    padded[seq, number] = q
    group = HEADS // keys
    columns = padded.view(seqs, most, keys, group, HEAD).permute(0, 2, 4, 3, 1).reshape(seqs, keys, HEAD, group * most)
    scores = (decoded("k", keys) @ columns).view(seqs, HEADS // group, length, group, most) * 0.125
    visible = lens.long()[:, None] + torch.arange(1, most + 1, device="cuda")
    hidden = torch.arange(length, device="cuda")[None, :, None] >= visible[:, None, :]
    scores = scores.masked_fill(hidden[:, None, :, None, :], float("-inf"))
    peak = scores.amax(dim=2, keepdim=True)
    weights = (scores - peak).exp()
    total = weights.sum(dim=2)
    # [seq][KV head][its query heads x rows][position] times the values.
    weights = weights.permute(0, 1, 3, 4, 2).reshape(seqs, KV_HEADS, HEADS // KV_HEADS * most, length)
    out = (weights @ decoded("v", KV_HEADS)).view(seqs, HEADS, most, HEAD)
    total, peak = total.view(seqs, HEADS, most), peak.view(seqs, HEADS, most)
    sink = 1.0 / (1.0 + (state["sinks"][None, :, None] - (peak + total.log())).exp())
    out = out / total[..., None] * sink[..., None]
    return {"out": out.transpose(1, 2)[seq, number]}


# -- the definitions, in 64 bits --------------------------------------------------
def _exact_linear4(case, make):
    out, inner, group, rows = case["out"], case["in"], case["group"], case["rows"]
    codes = make.codes(out, inner)
    scales = make.uniform(0.002, 0.008, out, -(-inner // group)).double()
    x = make.normal(rows, inner).double()
    residual = make.normal(rows, out).double() if case["epilogue"] == "ADD" else None
    if case["norm"]:
        x = x / torch.sqrt((x ** 2).sum(1, keepdim=True) / inner + EPS32)
    y = torch.zeros(rows, out, dtype=torch.float64, device="cuda")
    for g in range(scales.shape[1]):
        part = slice(g * group, min(inner, (g + 1) * group))
        y += (x[:, part] @ codes[:, part].double().t()) * scales[:, g]
    if case["epilogue"] == "GLU":
        return {"out": torch.relu(y[:, 0::2]) ** 2 * y[:, 1::2]}
    return {"out": y if residual is None else residual + y}


def _f32(x):
    """A 64-bit value rounded to FP32, as the row step and the codes are defined."""
    return x.float().double()


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


def _exact_block(rows):
    """What a block of rows [n][heads][64] (n up to 16) holds."""
    scale = _f32(rows.abs().amax(dim=2).amax(dim=0) / 127)
    inverse = _f32(1.0 / scale)
    return _f32(torch.round(_f32(rows * inverse[None, :, None])) * scale[None, :, None])


def _exact_pages(case, make):
    spans, keys = _spans(case), case["keys"]
    rows = sum(n for _, n in spans)
    open_rows = sum(length % BLOCK for length, _ in spans)
    if rows > 20000 or rows + open_rows > 16 * 2500:
        return None
    open_k, open_v = _unit_heads(make, open_rows, keys).double(), make.normal(open_rows, KV_HEADS, HEAD).double()
    qkv = make.normal(rows, (HEADS + 2 * KV_HEADS) * HEAD).double().view(rows, -1, HEAD)
    positions = torch.cat([torch.arange(length, length + n, device="cuda") for length, n in spans])
    rope = _factors(make, case, positions).double()
    source = torch.arange(keys, device="cuda") * KV_HEADS // keys
    turn = torch.arange(keys, device="cuda") * (HEADS // keys)
    q = _exact_rotate(qkv[:, :HEADS], rope)
    key, value = _exact_rotate(qkv[:, HEADS + source], rope[:, turn]), qkv[:, HEADS + KV_HEADS:]
    k, v, at, open_at = [], [], 0, 0
    for length, n in spans:
        held = length % BLOCK
        for result, earlier, new in ((k, open_k, key), (v, open_v, value)):
            whole = torch.cat([earlier[open_at:open_at + held], new[at:at + n]])
            result += [_exact_block(whole[b:b + BLOCK]) for b in range(0, held + n, BLOCK)]
        at, open_at = at + n, open_at + held
    return {"q": q, "k": torch.cat(k), "v": torch.cat(v)}


def _exact_attend(case, make):
    spans, keys = _spans(case), case["keys"]
    totals = [length + n for length, n in spans]
    k, v = _unit_heads(make, sum(totals), keys), make.normal(sum(totals), KV_HEADS, HEAD)
    q, sinks = _unit_heads(make, sum(n for _, n in spans), HEADS).double(), make.normal(HEADS).double()
    out, first, row = [], 0, 0
    for (length, n), total in zip(spans, totals):
        held = []
        for x in (k, v):
            x = x[first:first + total].double()
            pad = torch.zeros(-total % BLOCK, *x.shape[1:], dtype=torch.float64, device="cuda")
            blocks = torch.cat([x, pad]).view(-1, BLOCK, x.shape[1], HEAD)
            scale = _f32(blocks.abs().amax(dim=(1, 3), keepdim=True) / 127)
            codes = torch.round(_f32(blocks * _f32(1.0 / scale)))
            held.append((codes * scale).view(-1, x.shape[1], HEAD)[:total])
        key, value = (x.repeat_interleave(HEADS // x.shape[1], dim=1).transpose(0, 1).contiguous() for x in held)
        for r in range(n):
            seen = length + r + 1
            s = (key[:, :seen] @ q[row + r][:, :, None])[..., 0] / 8.0
            weights = torch.softmax(s, dim=1)
            sink = torch.sigmoid(torch.logsumexp(s, dim=1) - sinks)
            out.append((weights[:, None, :] @ value[:, :seen])[:, 0] * sink[:, None])
        first, row = first + total, row + n
    return {"out": torch.stack(out)}


def exact(case, seed):
    make = _Maker(seed)
    return {"linear4": _exact_linear4, "pages": _exact_pages, "attend": _exact_attend}[case["op"]](case, make)
