"""A serving step of models that norm their heads, rotate by several positions, keep their cache in 8 bits or
draft tokens as a tree, as cases that can be timed and compared:

- norms of queries and keys for each head with the position rotation (of one or several axes) in the same pass,
  alone ("turn") and with the step's keys and values into the paged cache ("append");
- the cache in 8 bits: quantised as it is written and read back ("quantise"), and the attention over it ("cached");
- attention of drafted tokens that form a tree over what is in the cache ("tree"), kept in 16 or in 8 bits.

Head layouts are those of the models the framework serves (32 and 40 heads of 128, 12 and 20 of 64), of image
encoders (16 of 80) and grouped ones.  A program that serves keeps its cache, the table of its pages, its index
tensors, its weights, its activation buffers and the views of them from step to step; that is what ``prepare`` makes.
``run`` is the operator's call, or the same in elementary torch operations (32 bits; angles, and what is quantised and
so lies next to a border, in 64; rounded once at the end).
"""
import math
import random

import torch

own = False

# (query heads, key and value heads, head dimension)
HEADS = ((32, 32, 128), (32, 8, 128), (40, 8, 128), (32, 4, 64), (20, 20, 64), (12, 12, 64), (16, 1, 128), (16, 16, 80),
         (24, 8, 96))
PAGES = (16, 32, 64, 128)
EPS = 1e-6
BASE = 10000.0


def _case(name, kind, heads, **more):
    c = {"name": name, "kind": kind, "heads": heads[0], "kv_heads": heads[1], "d": heads[2]}
    c.update(more)
    return c


def listed():
    return [
        # One generated token's queries, normed and turned, far into a long context: the smallest call.
        _case("turn_token", "turn", (32, 32, 128), rows=1, first=100003, rot=128, layout="halves", axes=1, grid=1, norm=True),
        # The patches of several images in an encoder: rotated by height and width, half of each head for either.
        _case("turn_patches", "turn", (16, 16, 80), rows=4097, first=0, rot=80, layout="halves", axes=2, grid=32, norm=True),
        # One step of 48 sequences that generate together: heads normed, queries and keys turned, keys and values to their pages.
        _case("append_tokens", "append", (32, 8, 128), sequences=48, rows_low=1, rows_high=1, past_low=0, past_high=4000,
              ragged=1, spare=0, page=16, order="tokens", rot=128, layout="halves", axes=1, grid=1, norm=True),
        # Four prompts with video frames in them: positions of time, height and width.
        _case("append_frames", "append", (32, 8, 128), sequences=4, rows_low=700, rows_high=2500, past_low=0, past_high=0,
              ragged=2, spare=5, page=64, order="heads", rot=128, layout="halves", axes=3, grid=24, norm=True),
        # The same step into a cache of 8 bits, and what it wrote read back, as where it moves to another machine.
        _case("quantise_tokens", "quantise", (32, 8, 128), sequences=64, rows_low=1, rows_high=1, past_low=0, past_high=3000,
              ragged=3, spare=0, page=16, order="heads", rot=128, layout="halves", axes=1, grid=1, norm=False),
        # Six prompts of different lengths into the cache of 8 bits at once, neighbours rotated.
        _case("quantise_prompts", "quantise", (40, 8, 128), sequences=6, rows_low=300, rows_high=2500, past_low=0, past_high=50,
              ragged=4, spare=3, page=32, order="tokens", rot=128, layout="pairs", axes=1, grid=1, norm=True),
        # One user's next token over a short context in 8 bits, every query head with its own keys.
        _case("cached_one_user", "cached", (32, 32, 128), sequences=1, rows_low=1, rows_high=1, chunk=0, past_low=776,
              past_high=776, ragged=5, spare=0, page=16, order="tokens"),
        # A step of 64 sequences of very different lengths, four query heads to a key head.
        _case("cached_batch", "cached", (32, 8, 128), sequences=64, rows_low=1, rows_high=1, chunk=0, past_low=3,
              past_high=4000, ragged=6, spare=0, page=16, order="heads"),
        # A long prompt's next piece over what is in the cache already: the largest computation.
        _case("cached_chunk", "cached", (32, 8, 128), sequences=1, rows_low=1, rows_high=1, chunk=1024, past_low=7001,
              past_high=7001, ragged=7, spare=0, page=64, order="heads"),
        # Eight sequences with very long contexts: the largest read.
        _case("cached_long", "cached", (40, 8, 128), sequences=8, rows_low=1, rows_high=1, chunk=0, past_low=50000,
              past_high=110000, ragged=8, spare=0, page=16, order="heads"),
        # One user's draft of 61 tokens over the cache in 16 bits.
        _case("tree_one_user", "tree", (32, 8, 128), sequences=1, rows_low=61, rows_high=61, chunk=0, past_low=2100,
              past_high=2100, ragged=9, spare=0, page=16, order="tokens", bits=16),
        # Small drafts of 24 sequences at once over a cache of 8 bits.
        _case("tree_batch", "tree", (32, 8, 128), sequences=24, rows_low=2, rows_high=13, chunk=0, past_low=10,
              past_high=6000, ragged=10, spare=2, page=32, order="heads", bits=8),
    ]


def _spread(rng, low, high):
    """An integer of [low, high], even over its logarithm."""
    if low < 1:
        return _spread(rng, low + 1, high + 1) - 1
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    kind = rng.choice(("turn", "append", "append", "quantise", "quantise", "cached", "cached", "cached", "cached", "tree",
                       "tree", "tree"))
    heads = rng.choice(HEADS)
    if kind in ("turn", "append", "quantise"):
        more = dict(rot=heads[2] // rng.choice((1, 1, 1, 2)), layout=rng.choice(("halves", "pairs")), axes=rng.choice((1, 1, 2, 3)),
                    grid=rng.randint(2, 40), norm=rng.choice((True, True, False)))
    if kind == "turn":
        return _unnamed(_case("", kind, heads, rows=_spread(rng, 1, 8192), first=_spread(rng, 0, 1 << 20), **more))
    common = {"ragged": rng.randrange(1 << 30), "spare": rng.choice((0, 0, 0, 1, 6)), "rows_low": 1, "rows_high": 1,
              "past_low": 0, "past_high": 0, "page": rng.choice(PAGES), "order": rng.choice(("tokens", "heads"))}
    if kind in ("append", "quantise"):
        common.update(more)
        if rng.random() < 0.5:
            common.update(sequences=_spread(rng, 1, 200), past_high=2000)
        else:
            common.update(sequences=_spread(rng, 1, 8), rows_high=_spread(rng, 2, 1500))
        return _unnamed(_case("", kind, heads, **common))
    common["chunk"] = 0
    most = 1 << 25  # values of keys in the cache, over all sequences
    if kind == "tree":
        common["bits"] = rng.choice((16, 8))
        common["rows_high"] = _spread(rng, 2, 100)
        common["rows_low"] = rng.choice((1, common["rows_high"]))
        common["sequences"] = _spread(rng, 1, max(1, 1024 // common["rows_high"]))
        longest = min(16384, most // (common["sequences"] * heads[1] * heads[2]) + 16)
    else:
        shape = rng.choice(("tokens", "tokens", "chunk", "mixed", "few"))
        if shape == "tokens":
            common.update(sequences=_spread(rng, 1, 128))
        elif shape == "chunk":
            common.update(sequences=1, chunk=_spread(rng, 17, 2048))
        elif shape == "mixed":
            common.update(sequences=_spread(rng, 2, 64), chunk=_spread(rng, 17, 1024))
        else:
            common.update(sequences=_spread(rng, 1, 32), rows_high=_spread(rng, 2, 16))
        longest = min(65536 if shape == "tokens" else 8192, most // (common["sequences"] * heads[1] * heads[2]) + 16)
    common["past_high"] = _spread(rng, 1, longest)
    common["past_low"] = rng.choice((0, common["past_high"] // 2, common["past_high"]))
    return _unnamed(_case("", kind, heads, **common))


def _unnamed(case):
    del case["name"]
    return case


def _sequences(case):
    """(new rows, keys with them) of each sequence."""
    g = random.Random(case["ragged"])
    out = []
    for i in range(case["sequences"]):
        rows = case["chunk"] if case.get("chunk") and i == 0 else g.randint(case["rows_low"], case["rows_high"])
        out.append((rows, rows + g.randint(case["past_low"], case["past_high"])))
    return out


def _starts(counts):
    at = [0]
    for c in counts:
        at.append(at[-1] + c)
    return at


def _trees(case):
    """For each sequence, for each drafted token the set of drafted tokens that it follows, itself among them, as bits:
    each follows an earlier one (the likelier ones more often), the first what is in the cache."""
    g = random.Random(case["ragged"] + 1)
    out = []
    for rows, _ in _sequences(case):
        seen = [1]
        for j in range(1, rows):
            seen.append(seen[int(j * g.random() ** 2)] | 1 << j)
        out.append(seen)
    return out


# ---- positions ---------------------------------------------------------------------------------------

def _sections(case):
    """Rotated pairs of each axis: equal parts, the first with what is left over."""
    pairs, axes = case["rot"] // 2, case["axes"]
    return [pairs - (axes - 1) * (pairs // axes)] + [pairs // axes] * (axes - 1)


def _positions(case, rows, first):
    """[axes][rows] of rows from `first` on: text counts on; a grid counts frames, lines and columns."""
    if case["axes"] == 1:
        return [list(range(first, first + rows))]
    w = case["grid"]
    axes = [[first + i // (w * w) for i in range(rows)], [first + i // w % w for i in range(rows)], [first + i % w for i in range(rows)]]
    return axes[-case["axes"]:]


def _rotated(x, s):
    """x [rows, heads, d], of its own bits, with its first columns turned by the rows' angles."""
    case, rows = s["case"], x.shape[0]
    angle = s["positions"][s["axis"]][:, :rows].t().double() * s["frequencies"]
    cos, sin = (f(angle).to(x.dtype)[:, None, :] for f in (torch.cos, torch.sin))
    rot = case["rot"]
    if case["layout"] == "halves":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos), dim=-1)
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), dim=-1).flatten(-2)
    return torch.cat((turned, x[..., rot:]), dim=-1)


def _normed(x, weight):
    """Each head of x [rows, heads, d], of its own bits, by its root mean square, times the weight."""
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.to(x.dtype)


# ---- inputs --------------------------------------------------------------------------------------------

def _inputs(case, seed):
    """The tensors of a case, made from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, heads, kv, d = case["kind"], case["heads"], case["kv_heads"], case["d"]

    def normal(*shape):
        return torch.randn(*shape, dtype=torch.float16, device="cuda", generator=g)

    def zeros(*shape):
        return torch.zeros(*shape, dtype=torch.float16, device="cuda")

    def ints(values):
        return torch.tensor(values, dtype=torch.int32).cuda()

    s = {"case": case}
    if kind in ("turn", "append", "quantise"):
        s["q_weight"], s["k_weight"] = ((1 + 0.2 * normal(d).float()).half() for _ in range(2))
    if kind == "turn":
        rows = case["rows"]
        s["q"], s["out"] = 3 * normal(rows, heads, d), zeros(rows, heads, d)
        s["positions"] = ints(_positions(case, rows, case["first"]))
        return s
    seqs = _sequences(case)
    rows, lengths = [r for r, _ in seqs], [n for _, n in seqs]
    starts, total = _starts(rows), sum(rows) + case["spare"]
    s.update(seqs=seqs, starts=starts, row_offsets=ints(starts), lengths=ints(lengths), out=zeros(total, heads, d))
    page = case["page"]
    need = [(n + page - 1) // page for n in lengths]
    pages = sum(need) + 3  # (some pages belong to nobody)
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(len(seqs), max(need) + 1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    s["table"] = table
    by_tokens = case["order"] == "tokens"
    if kind == "append" or case.get("bits") == 16:
        for t in ("key_pages", "value_pages"):
            s[t] = normal(pages, page, kv, d).permute(0, 2, 1, 3) if by_tokens else normal(pages, kv, page, d)
    else:
        for t in ("key_codes", "value_codes"):  # (codes of normal values with their largest at 3.5 deviations)
            codes = torch.empty(pages, page * kv * d, dtype=torch.uint8, device="cuda")
            for p in range(0, pages, 4096):
                codes[p:p + 4096] = (normal(min(4096, pages - p), page * kv * d).float() * 36.4 + 127.5).clamp(0, 255).to(torch.uint8)
            s[t] = codes.view(pages, page, kv, d).permute(0, 2, 1, 3) if by_tokens else codes.view(pages, kv, page, d)
        for t in ("key_scales", "value_scales"):
            scales = (torch.rand(pages, page * kv, device="cuda", generator=g) * 0.01 + 0.02).half()
            s[t] = scales.view(pages, page, kv).permute(0, 2, 1) if by_tokens else scales.view(pages, kv, page)
    if kind in ("append", "quantise"):
        qkv = 2 * normal(total, heads + 2 * kv, d)
        s["q"], s["k"], s["v"] = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
        positions = [[], [], []][:case["axes"]]
        for r, n in seqs:
            for axis, p in zip(positions, _positions(case, r, n - r)):
                axis += p
        s["positions"] = ints([axis + [0] * case["spare"] for axis in positions])
        if kind == "quantise":
            s["key_out"], s["value_out"] = zeros(total, kv, d), zeros(total, kv, d)
    else:
        s["q"] = normal(total, heads, d)
    if kind == "tree":
        words = (max(rows) + 31) // 32
        bits = [[(seen >> 32 * w & 0xffffffff) - (seen >> 32 * w + 31 & 1) * (1 << 32) for w in range(words)]
                for tree in _trees(case) for seen in tree]
        s["tree_bits"] = ints(bits + [[0] * words] * case["spare"])
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["scale"] = 1.5 / math.sqrt(case["d"])
    turned = case["kind"] in ("turn", "append", "quantise")
    if not own:
        if turned:
            rot = case["rot"]
            s["frequencies"] = (BASE ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)).cuda()
            s["axis"] = torch.tensor([a for a, n in enumerate(_sections(case)) for _ in range(n)]).cuda()
        return s
    from adrastea_amd import (DraftTree, GpuKernels, HeadNorm, PagedBatch, PagedCache, PagedCacheU8, RotaryAxes, RotaryLayout,
                              TensorView)
    s["kernels"] = GpuKernels()
    for t in ("q", "k", "v", "out", "key_out", "value_out"):  # the operators take [heads, rows, d] views
        if t in s:
            s[t + "_view"] = TensorView.of(s[t].permute(1, 0, 2))
    if turned:
        layout = {"halves": RotaryLayout.HALVES, "pairs": RotaryLayout.PAIRS}[case["layout"]]
        s["rotary"] = RotaryAxes.new(case["rot"], _sections(case), base=BASE, layout=layout)
        s["q_norm"] = HeadNorm(s["q_weight"], EPS) if case["norm"] else None
        s["k_norm"] = HeadNorm(s["k_weight"], EPS) if case["norm"] else None
    if "key_pages" in s:
        s["cache"] = PagedCache(TensorView.of(s["key_pages"]), TensorView.of(s["value_pages"]))
    if "key_codes" in s:
        s["cache"] = PagedCacheU8(*(TensorView.of(s[t]) for t in ("key_codes", "key_scales", "value_codes", "value_scales")))
    if "seqs" in s:
        s["batch"] = PagedBatch(s["row_offsets"], s["lengths"], s["table"], max(r for r, _ in s["seqs"]),
                                max(n for _, n in s["seqs"]))
    if "tree_bits" in s:
        s["tree"] = DraftTree(s["tree_bits"])
    return s


# ---- one pass --------------------------------------------------------------------------------------------

def run(s):
    case, kind = s["case"], s["case"]["kind"]
    if own:
        k = s["kernels"]
        if kind == "turn":
            k.norm_rotary_f16(s["out_view"], s["q_view"], s["positions"], s["rotary"], s["q_norm"])
        elif kind == "append":
            k.append_norm_f16(s["cache"], s["batch"], s["k_view"], s["v_view"], s["rotary"], s["out_view"], s["q_view"],
                              s["positions"], s["q_norm"], s["k_norm"])
            return s["out"], s["key_pages"], s["value_pages"]
        elif kind == "quantise":
            k.append_u8(s["cache"], s["batch"], s["k_view"], s["v_view"], s["rotary"], s["out_view"], s["q_view"],
                        s["positions"], s["q_norm"], s["k_norm"])
            k.read_u8(s["key_out_view"], s["value_out_view"], s["cache"], s["batch"])
            return s["out"], s["key_out"], s["value_out"]
        elif kind == "cached":
            k.attention_paged_u8(s["out_view"], s["q_view"], s["cache"], s["batch"], s["scale"])
        elif case["bits"] == 16:
            k.attention_tree_f16(s["out_view"], s["q_view"], s["cache"], s["batch"], s["tree"], s["scale"])
        else:
            k.attention_tree_u8(s["out_view"], s["q_view"], s["cache"], s["batch"], s["tree"], s["scale"])
        return s["out"]
    if kind in ("turn", "append", "quantise"):
        rows = s["starts"][-1] if "starts" in s else case["rows"]
        q = s["q"][:rows].float()
        s["out"][:rows] = _rotated(_normed(q, s["q_weight"]) if case["norm"] else q, s).half()
        if kind == "turn":
            return s["out"]
        key = s["k"][:rows].double() if kind == "quantise" else s["k"][:rows].float()
        key = _rotated(_normed(key, s["k_weight"]) if case["norm"] else key, s)
        index = torch.arange(rows, device="cuda")
        seq = torch.searchsorted(s["row_offsets"][1:].contiguous(), index.to(torch.int32), right=True)
        at = s["lengths"][seq] - s["row_offsets"][seq + 1] + index
        pages, slots = s["table"][seq, at // case["page"]].long(), at % case["page"]
        if kind == "append":
            s["key_pages"][pages, :, slots] = key.half()
            s["value_pages"][pages, :, slots] = s["v"][:rows]
            return s["out"], s["key_pages"], s["value_pages"]
        for t, x in (("key", key), ("value", s["v"][:rows].double())):
            codes, scales = _quantised(x)
            s[t + "_codes"][pages, :, slots], s[t + "_scales"][pages, :, slots] = codes, scales
            s[t + "_out"][:rows] = _value_of(s[t + "_codes"][pages, :, slots], s[t + "_scales"][pages, :, slots]).half()
        return s["out"], s["key_out"], s["value_out"]
    trees = _trees(case) if kind == "tree" else None
    for i, (rows, length) in enumerate(s["seqs"]):
        first = s["starts"][i]
        key, value = (_from_pages(s, t, i, length) for t in ("key", "value"))
        drafted = s["tree_bits"][first:first + rows] if trees else None
        s["out"][first:first + rows] = _plain_attention(s["q"][first:first + rows].float(), key, value, s["scale"], drafted)
    return s["out"]


def _quantised(x):
    """x [rows, heads, d] in 64 bits as codes and one scale for each head: code c stands for (c - 127.5) scale, and the
    scale is the largest |x| / 127.5 rounded up to 16 bits (513.5 at most, so that all codes' values are finite in 16)."""
    exact = x.abs().amax(-1) / 127.5
    scale = exact.half()
    up = torch.nextafter(scale, torch.full_like(scale, math.inf))
    scale = torch.where(scale.double() < exact, up, scale).clamp(max=513.5)
    codes = torch.floor(x / torch.where(scale == 0, 1, scale.double())[..., None]) + 128
    return codes.clamp(0, 255).to(torch.uint8), scale


def _value_of(codes, scales):
    return (codes.float() - 127.5) * scales.float()[..., None]


def _from_pages(s, name, i, length):
    """[kv heads, length, d] of one sequence, in 32 bits."""
    page = s["case"]["page"]
    pages = s["table"][i, :(length + page - 1) // page].long()
    picked = (s[name + "_pages"][pages].float() if name + "_pages" in s else
              _value_of(s[name + "_codes"][pages], s[name + "_scales"][pages]))
    return picked.permute(1, 0, 2, 3).flatten(1, 2)[:, :length]


def _plain_attention(q, key, value, scale, drafted):
    """q [rows, heads, d], key and value [kv heads, keys, d], 32 bits; causal from the last key on, or the last keys as
    the rows' bits say."""
    (rows, heads, d), (kv, n, _) = q.shape, key.shape
    group = heads // kv
    hidden = torch.arange(n, device="cuda") > torch.arange(rows, device="cuda")[:, None] + (n - rows)
    if drafted is not None:
        j = torch.arange(rows, device="cuda")
        hidden = torch.zeros_like(hidden)
        hidden[:, n - rows:] = (drafted[:, j // 32] >> (j % 32) & 1) == 0
    hidden = hidden.repeat(group, 1)
    q = q.view(rows, kv, group, d).permute(1, 2, 0, 3).reshape(kv, group * rows, d)
    step = kv if kv * group * rows * n < 1 << 28 else 1  # (heads at a time)
    out = []
    for h in range(0, kv, step):
        scores = torch.bmm(q[h:h + step], key[h:h + step].transpose(1, 2).contiguous()).mul_(scale)
        scores.masked_fill_(hidden, float("-inf"))
        weights = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
        total = weights.sum(-1, keepdim=True)
        out.append(torch.bmm(weights, value[h:h + step].contiguous()) / total)
    return torch.cat(out).view(kv, group, rows, d).permute(2, 0, 1, 3).reshape(rows, heads, d).half()


# ---- what a pass cannot do without --------------------------------------------------------------------------

def work(case):
    heads, kv, d = case["heads"], case["kv_heads"], case["d"]
    if case["kind"] == "turn":
        values = case["rows"] * heads * d
        return {"bytes": 4 * values + 4 * case["axes"] * case["rows"], "flops": (7 if case["norm"] else 3) * values}
    seqs = _sequences(case)
    rows, keys = sum(r for r, _ in seqs), sum(n for _, n in seqs)
    if case["kind"] == "append":
        return {"bytes": 4 * rows * (heads + 2 * kv) * d, "flops": 7 * rows * (heads + kv) * d}
    if case["kind"] == "quantise":  # (codes and scales are written, and 16 bits for them)
        return {"bytes": rows * (4 * heads * d + 2 * kv * (2 * d + d + 2 + 2 * d)),
                "flops": rows * d * (7 * heads + 15 * kv)}
    if case["kind"] == "cached":
        pairs = sum(r * n - r * (r - 1) // 2 for r, n in seqs)
    else:
        pairs = sum(r * (n - r) for r, n in seqs) + sum(bin(seen).count("1") for tree in _trees(case) for seen in tree)
    value_bytes = 2 * d if case.get("bits") == 16 else d + 2
    return {"bytes": 4 * rows * heads * d + 2 * keys * kv * value_bytes, "flops": 4 * pairs * heads * d}


# ---- the definition, in 64 bits -------------------------------------------------------------------------------

def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "turn":
        return _turned_exactly(case, s["q"], s["positions"], s["q_weight"])
    out = s["out"].double()
    if case["kind"] in ("append", "quantise"):
        rows = s["starts"][-1]
        turned = {"q": _turned_exactly(case, s["q"][:rows], s["positions"], s["q_weight"]),
                  "key": _turned_exactly(case, s["k"][:rows], s["positions"], s["k_weight"]), "value": s["v"][:rows].double()}
        out[:rows] = turned["q"]
        if case["kind"] == "quantise":
            read = []
            for t in ("key", "value"):
                whole = s[t + "_out"].double()
                whole[:rows] = _through_8_bits(turned[t])
                read.append(whole)
            return (out, *read)
        pages = [s[t + "_pages"].double() for t in ("key", "value")]
        for i, (new, length) in enumerate(s["seqs"]):
            first, past = s["starts"][i], length - new
            for page in range(past // case["page"], (length - 1) // case["page"] + 1):
                low, high = max(past, page * case["page"]), min(length, (page + 1) * case["page"])
                slots = slice(low - page * case["page"], high - page * case["page"])
                for t, pool in zip(("key", "value"), pages):
                    pool[int(s["table"][i, page]), :, slots] = turned[t][first + low - past:first + high - past].permute(1, 0, 2)
        return (out, *pages)
    scale, group = 1.5 / math.sqrt(case["d"]), case["heads"] // case["kv_heads"]
    trees = _trees(case) if case["kind"] == "tree" else None
    for i, (rows, length) in enumerate(s["seqs"]):
        first, past = s["starts"][i], length - rows
        used = s["table"][i, :-(-length // case["page"])].tolist()
        if trees:
            seen = torch.tensor([[tree >> j & 1 for j in range(rows)] for tree in trees[i]], dtype=torch.bool).cuda()
        for h in range(case["kv_heads"]):
            key, value = (_whole_exactly(s, t, h, used)[:length] for t in ("key", "value"))
            columns = torch.arange(length, device="cuda")
            for low in range(0, rows, 2048):
                high = min(rows, low + 2048)
                last = torch.arange(low, high, device="cuda") + past
                visible = columns[None, :] <= last[:, None]
                if trees:
                    visible = torch.ones_like(visible)
                    visible[:, past:] = seen[low:high]
                for e in range(h * group, (h + 1) * group):
                    scores = s["q"][first + low:first + high, e].double() @ key.t() * scale
                    scores = torch.where(visible, scores, -torch.inf)
                    weights = torch.exp(scores - torch.logsumexp(scores, dim=1, keepdim=True))
                    out[first + low:first + high, e] = weights @ value
    return out


def _whole_exactly(s, name, h, used):
    """[keys, d] of one key head on the pages `used`."""
    d = s["case"]["d"]
    if name + "_pages" in s:
        return s[name + "_pages"][:, h][used].reshape(-1, d).double()
    codes, scales = s[name + "_codes"][:, h][used].reshape(-1, d), s[name + "_scales"][:, h][used].reshape(-1)
    return (2 * codes.double() - 255) * (scales.double() / 2)[:, None]


def _through_8_bits(x):
    """What the codes of x [rows, heads, d] stand for: the middle of the step of x, steps counted from zero."""
    most = x.abs().max(dim=-1, keepdim=True).values / 127.5
    # (the numbers of 16 bits at or above: a mantissa of 11 bits, from 2^-14 on, in steps of 2^-24 below)
    unit = torch.ldexp(torch.ones_like(most), torch.frexp(most.clamp(min=2.0 ** -14)).exponent - 11)
    step = (torch.ceil(most / unit) * unit).clamp(max=513.5)
    n = torch.where(step > 0, torch.floor(x / torch.where(step > 0, step, 1.0)), 0.0).clamp(-128, 127)
    return (n + 0.5) * step


def _turned_exactly(case, x, positions, weight):
    """x [rows, heads, d] normed and turned as complex numbers, one pair of columns after the other."""
    out, rows = x.double(), x.shape[0]
    if case["norm"]:
        out = out / torch.sqrt(out.square().sum(dim=-1, keepdim=True) / case["d"] + EPS) * weight.double()
    rot, half, pair = case["rot"], case["rot"] // 2, 0
    for axis, count in enumerate(_sections(case)):
        for _ in range(count):
            angle = positions[axis, :rows].double() * BASE ** (-2.0 * pair / rot)
            a, b = (pair, pair + half) if case["layout"] == "halves" else (2 * pair, 2 * pair + 1)
            turned = torch.complex(out[..., a], out[..., b]) * torch.polar(torch.ones_like(angle), angle)[:, None]
            out[..., a], out[..., b] = turned.real, turned.imag
            pair += 1
    return out
