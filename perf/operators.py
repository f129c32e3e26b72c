"""Serving several sequences at once: rotary positions, the paged cache that a step fills, and the
attention that reads it or reads whole prompts packed behind each other, as cases that can be timed
and compared.

Head layouts are those of the models the framework serves (32 and 40 heads of 128, 12 and 20 of 64)
and grouped ones, in which several query heads share a key and value head.  A program that serves
keeps its cache, the table of its pages, its index tensors, its activation buffers and the views of
them from step to step; that is what ``prepare`` makes.  ``run`` is the operator's call, or the same in
elementary torch operations (32 bits, angles in 64, rounded once at the end).
"""
import math
import random

import torch

own = False

# (query heads, key and value heads, head dimension)
HEADS = ((32, 32, 128), (32, 8, 128), (40, 8, 128), (32, 4, 64), (20, 20, 64), (12, 12, 64), (16, 1, 128))
PAGES = (16, 32, 64, 128)


def _case(name, kind, heads, **more):
    c = {"name": name, "kind": kind, "heads": heads[0], "kv_heads": heads[1], "d": heads[2]}
    c.update(more)
    return c


def listed():
    return [
        # The rotation of one generated token's queries, far into a long context: the smallest call.
        _case("rotary_token", "rotary", (32, 32, 128), rows=1, first=100003, rot=128, layout="halves", scaling="none"),
        # Queries of a prompt of odd length, neighbours rotated, half of each head, positions
        # stretched by four.
        _case("rotary_prompt_pairs", "rotary", (40, 8, 128), rows=4099, first=0, rot=64, layout="pairs", scaling="linear"),
        # One step of 48 sequences that generate together: queries rotated, keys and values to their pages.
        _case("append_tokens", "append", (32, 8, 128), sequences=48, rows_low=1, rows_high=1, chunk=0, past_low=0,
              past_high=4000, ragged=1, spare=0, page=16, order="tokens", rot=128, layout="halves", scaling="wavelength"),
        # Four prompts of different lengths into the cache at once, from one fused projection.
        _case("append_prompts", "append", (32, 8, 128), sequences=4, rows_low=700, rows_high=2500, chunk=0, past_low=0,
              past_high=0, ragged=2, spare=5, page=64, order="heads", rot=128, layout="halves", scaling="yarn"),
        # One user's next token over a short context, every query head with its own keys.
        _case("paged_one_user", "paged", (32, 32, 128), sequences=1, rows_low=1, rows_high=1, chunk=0, past_low=776,
              past_high=776, ragged=3, spare=0, page=16, order="tokens"),
        # A step of 64 sequences of very different lengths, four query heads to a key head.
        _case("paged_batch", "paged", (32, 8, 128), sequences=64, rows_low=1, rows_high=1, chunk=0, past_low=3,
              past_high=4000, ragged=4, spare=0, page=16, order="tokens"),
        # A long prompt's next piece over what is in the cache already.
        _case("paged_chunk", "paged", (32, 8, 128), sequences=1, rows_low=1, rows_high=1, chunk=1024, past_low=7001,
              past_high=7001, ragged=5, spare=0, page=64, order="heads"),
        # A prompt's piece and the tokens of 40 others in one step, heads of 64.
        _case("paged_mixed", "paged", (32, 4, 64), sequences=41, rows_low=1, rows_high=1, chunk=500, past_low=1,
              past_high=2500, ragged=6, spare=4, page=32, order="tokens"),
        # Eight sequences with very long contexts: the largest read.
        _case("paged_long", "paged", (40, 8, 128), sequences=8, rows_low=1, rows_high=1, chunk=0, past_low=50000,
              past_high=110000, ragged=7, spare=0, page=16, order="tokens"),
        # Sixteen short prompts packed, 12 heads of 64 as in a text encoder.
        _case("packed_short", "packed", (12, 12, 64), sequences=16, rows_low=5, rows_high=77, chunk=0, past_low=0,
              past_high=0, ragged=8, spare=0),
        # Prompts of very different lengths in one call.
        _case("packed_prompts", "packed", (32, 8, 128), sequences=9, rows_low=100, rows_high=4000, chunk=0, past_low=0,
              past_high=0, ragged=9, spare=7),
        # One long prompt: the largest computation.
        _case("packed_long", "packed", (32, 8, 128), sequences=1, rows_low=1, rows_high=1, chunk=16384, past_low=0,
              past_high=0, ragged=10, spare=0),
    ]


def _spread(rng, low, high):
    """An integer of [low, high], even over its logarithm."""
    if low < 1:
        return _spread(rng, low + 1, high + 1) - 1
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    kind = rng.choice(("rotary", "append", "append", "paged", "paged", "paged", "paged", "packed", "packed", "packed"))
    heads = rng.choice(HEADS)
    if kind == "rotary":
        rot = heads[2] // rng.choice((1, 1, 2, 4))
        return _unnamed(_case("", kind, heads, rows=_spread(rng, 1, 8192), first=_spread(rng, 0, 1 << 20), rot=rot,
                              layout=rng.choice(("halves", "pairs")),
                              scaling=rng.choice(("none", "linear", "wavelength", "yarn"))))
    cache = {"page": rng.choice(PAGES), "order": rng.choice(("tokens", "heads"))} if kind != "packed" else {}
    common = {"ragged": rng.randrange(1 << 30), "spare": rng.choice((0, 0, 0, 1, 6)), "chunk": 0, "rows_low": 1,
              "rows_high": 1, "past_low": 0, "past_high": 0, **cache}
    if kind == "append":
        common.update(rot=heads[2] // rng.choice((1, 1, 2)), layout=rng.choice(("halves", "pairs")),
                      scaling=rng.choice(("none", "linear", "wavelength", "yarn")))
        if rng.random() < 0.5:
            common.update(sequences=_spread(rng, 1, 200), past_high=2000)
        else:
            common.update(sequences=_spread(rng, 1, 8), rows_high=_spread(rng, 2, 1500))
    elif kind == "paged":
        shape = rng.choice(("tokens", "tokens", "chunk", "mixed", "few"))
        most = 1 << 25  # values of keys in the cache, over all sequences
        if shape == "tokens":
            common.update(sequences=_spread(rng, 1, 128))
        elif shape == "chunk":
            common.update(sequences=1, chunk=_spread(rng, 17, 2048))
        elif shape == "mixed":
            common.update(sequences=_spread(rng, 2, 64), chunk=_spread(rng, 17, 1024))
        else:
            common.update(sequences=_spread(rng, 1, 32), rows_high=_spread(rng, 2, 16))
        longest = min(65536 if shape == "tokens" else 16384, most // (common["sequences"] * heads[1] * heads[2]) + 16)
        common["past_high"] = _spread(rng, 1, longest)
        common["past_low"] = rng.choice((0, common["past_high"] // 2, common["past_high"]))
    else:
        common.update(sequences=_spread(rng, 1, 32))
        common["rows_high"] = _spread(rng, 1, min(8192, 24576 // common["sequences"]))
        common["rows_low"] = rng.choice((1, common["rows_high"]))
        common["past_high"] = rng.choice((0, 0, 100))
    return _unnamed(_case("", kind, heads, **common))


def _unnamed(case):
    del case["name"]
    return case


def _sequences(case):
    """(new rows, keys with them) of each sequence."""
    g = random.Random(case["ragged"])
    out = []
    for i in range(case["sequences"]):
        rows = case["chunk"] if case["chunk"] and i == 0 else g.randint(case["rows_low"], case["rows_high"])
        out.append((rows, rows + g.randint(case["past_low"], case["past_high"])))
    return out


def _starts(counts):
    at = [0]
    for c in counts:
        at.append(at[-1] + c)
    return at


# ---- positions ---------------------------------------------------------------------------------------

BASE = 10000.0
LINEAR = 4.0
WAVELENGTH = {"factor": 8.0, "low": 1.0, "high": 4.0, "original": 8192}
YARN = {"factor": 4.0, "original": 4096, "fast": 32.0, "slow": 1.0}


def _frequencies(case):
    """Radians a position for each rotated pair, in 64 bits, and the magnitude of the rotated values."""
    rot, scaling = case["rot"], case["scaling"]
    f = BASE ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    if scaling == "linear":
        return f / LINEAR, 1.0
    if scaling == "wavelength":
        w = WAVELENGTH
        turns = w["original"] * f / (2 * math.pi)
        keep = ((turns - w["low"]) / (w["high"] - w["low"])).clamp(0, 1)
        return f * keep + f / w["factor"] * (1 - keep), 1.0
    if scaling == "yarn":
        y = YARN

        def index(turns):
            return rot * math.log(y["original"] / (turns * 2 * math.pi)) / (2 * math.log(BASE))
        low, high = max(math.floor(index(y["fast"])), 0), min(math.ceil(index(y["slow"])), rot - 1)
        ramp = ((torch.arange(rot // 2, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0, 1)
        return f * (1 - ramp) + f / y["factor"] * ramp, 0.1 * math.log(y["factor"]) + 1.0
    return f, 1.0


def _rotary_handle(case):
    from adrastea_amd import Rotary, RotaryLayout, RotaryScaling
    scaling = {"none": RotaryScaling.Identity(), "linear": RotaryScaling.Linear(LINEAR),
               "wavelength": RotaryScaling.Wavelength(WAVELENGTH["factor"], WAVELENGTH["low"], WAVELENGTH["high"],
                                                      WAVELENGTH["original"]),
               "yarn": RotaryScaling.Yarn(YARN["factor"], YARN["original"], YARN["fast"], YARN["slow"])}[case["scaling"]]
    layout = {"halves": RotaryLayout.HALVES, "pairs": RotaryLayout.PAIRS}[case["layout"]]
    return Rotary.new(case["rot"], base=BASE, layout=layout, scaling=scaling)


def _rotated(x, positions, frequencies, magnitude, layout):
    """x [rows, heads, d] in 32 bits with its first columns turned by the rows' angles."""
    angle = positions.double()[:, None] * frequencies
    cos, sin = ((f(angle) * magnitude).float()[:, None, :] for f in (torch.cos, torch.sin))
    rot = 2 * frequencies.numel()
    if layout == "halves":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos), dim=-1)
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), dim=-1).flatten(-2)
    return torch.cat((turned, x[..., rot:]), dim=-1)


# ---- inputs --------------------------------------------------------------------------------------------

def _inputs(case, seed):
    """The tensors of a case, made from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, heads, kv, d = case["kind"], case["heads"], case["kv_heads"], case["d"]

    def normal(*shape):
        return torch.randn(*shape, dtype=torch.float16, device="cuda", generator=g)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32).cuda()

    if kind == "rotary":
        rows = case["rows"]
        return {"x": normal(rows, heads, d), "out": torch.zeros(rows, heads, d, dtype=torch.float16, device="cuda"),
                "positions": ints(range(case["first"], case["first"] + rows))}
    seqs = _sequences(case)
    rows, lengths = [r for r, _ in seqs], [n for _, n in seqs]
    starts, total = _starts(rows), sum(rows) + case["spare"]
    s = {"seqs": seqs, "starts": starts, "row_offsets": ints(starts)}
    s["out"] = torch.zeros(total, heads, d, dtype=torch.float16, device="cuda")
    if kind == "packed":
        s["key_starts"] = _starts(lengths)
        s["key_offsets"] = ints(s["key_starts"])
        if rows == lengths:  # whole prompts: one fused projection
            qkv = normal(total, heads + 2 * kv, d)
            s["q"], s["k"], s["v"] = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
        else:
            s["q"], s["k"], s["v"] = normal(total, heads, d), normal(sum(lengths), kv, d), normal(sum(lengths), kv, d)
        return s
    page = case["page"]
    need = [(n + page - 1) // page for n in lengths]
    pages = sum(need) + 3  # (some pages belong to nobody)
    shape = (pages, page, kv, d) if case["order"] == "tokens" else (pages, kv, page, d)
    s["key_pages"], s["value_pages"] = normal(*shape), normal(*shape)
    if case["order"] == "tokens":
        s["key_pages"], s["value_pages"] = (s[t].permute(0, 2, 1, 3) for t in ("key_pages", "value_pages"))
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(len(seqs), max(need) + 1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    s["table"], s["lengths"] = table, ints(lengths)
    if kind == "append":
        qkv = normal(total, heads + 2 * kv, d)
        s["q"], s["k"], s["v"] = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    else:
        s["q"] = normal(total, heads, d)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"], s["scale"] = case, 1.5 / math.sqrt(case["d"])
    if not own:
        if case["kind"] in ("rotary", "append"):
            f, s["magnitude"] = _frequencies(case)
            s["frequencies"] = f.cuda()
        return s
    from adrastea_amd import GpuKernels, PackedBatch, PagedBatch, PagedCache, TensorView
    s["kernels"] = GpuKernels()
    for t in ("x", "q", "k", "v", "out"):  # the operators take [heads, rows, d] views
        if t in s:
            s[t + "_view"] = TensorView.of(s[t].permute(1, 0, 2))
    if case["kind"] in ("rotary", "append"):
        s["rotary"] = _rotary_handle(case)
    if case["kind"] in ("append", "paged"):
        s["cache"] = PagedCache(TensorView.of(s["key_pages"]), TensorView.of(s["value_pages"]))
        s["batch"] = PagedBatch(s["row_offsets"], s["lengths"], s["table"], max(r for r, _ in s["seqs"]),
                                max(n for _, n in s["seqs"]))
    if case["kind"] == "packed":
        s["batch"] = PackedBatch(s["row_offsets"], s["key_offsets"], max(r for r, _ in s["seqs"]),
                                 max(n for _, n in s["seqs"]))
    return s


# ---- one pass --------------------------------------------------------------------------------------------

def run(s):
    kind = s["case"]["kind"]
    if own:
        k = s["kernels"]
        if kind == "rotary":
            k.rotary_f16(s["out_view"], s["x_view"], s["positions"], s["rotary"])
        elif kind == "append":
            k.append_f16(s["cache"], s["batch"], s["k_view"], s["v_view"], s["rotary"], s["out_view"], s["q_view"])
            return s["out"], s["key_pages"], s["value_pages"]
        elif kind == "paged":
            k.attention_paged_f16(s["out_view"], s["q_view"], s["cache"], s["batch"], s["scale"])
        else:
            k.attention_packed_f16(s["out_view"], s["q_view"], s["k_view"], s["v_view"], s["batch"], s["scale"])
        return s["out"]
    if kind == "rotary":
        s["out"].copy_(_rotated(s["x"].float(), s["positions"], s["frequencies"], s["magnitude"], s["case"]["layout"]))
        return s["out"]
    if kind == "append":
        _plain_append(s)
        return s["out"], s["key_pages"], s["value_pages"]
    for i, (rows, length) in enumerate(s["seqs"]):
        first = s["starts"][i]
        q = s["q"][first:first + rows].float()
        if kind == "paged":
            key, value = (_from_pages(s, t, i, length).float() for t in ("key_pages", "value_pages"))
        else:
            at = s["key_starts"][i]
            key, value = (s[t][at:at + length].permute(1, 0, 2).float() for t in ("k", "v"))
        s["out"][first:first + rows] = _plain_attention(q, key, value, s["scale"])
    return s["out"]


def _from_pages(s, name, i, length):
    """[kv heads, length, d] of one sequence."""
    page = s["case"]["page"]
    picked = s[name][s["table"][i, :(length + page - 1) // page].long()]
    return picked.permute(1, 0, 2, 3).flatten(1, 2)[:, :length]


def _plain_append(s):
    case = s["case"]
    page, rows = case["page"], s["starts"][-1]
    index = torch.arange(rows, device="cuda")
    seq = torch.searchsorted(s["row_offsets"][1:].contiguous(), index.to(torch.int32), right=True)
    at = s["lengths"][seq] - s["row_offsets"][seq + 1] + index
    turn = (at, s["frequencies"], s["magnitude"], case["layout"])
    s["out"][:rows] = _rotated(s["q"][:rows].float(), *turn).half()
    pages, slots = s["table"][seq, at // page].long(), at % page
    s["key_pages"][pages, :, slots] = _rotated(s["k"][:rows].float(), *turn).half()
    s["value_pages"][pages, :, slots] = s["v"][:rows]


def _plain_attention(q, key, value, scale):
    """q [rows, heads, d], key and value [kv heads, keys, d], 32 bits; causal from the last key on."""
    (rows, heads, d), (kv, n, _) = q.shape, key.shape
    group = heads // kv
    hidden = torch.arange(n, device="cuda") > torch.arange(rows, device="cuda")[:, None] + (n - rows)
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
    if case["kind"] == "rotary":
        values = case["rows"] * heads * d
        return {"bytes": 4 * values + 4 * case["rows"], "flops": 3 * case["rows"] * heads * case["rot"]}
    seqs = _sequences(case)
    rows, keys = sum(r for r, _ in seqs), sum(n for _, n in seqs)
    if case["kind"] == "append":
        return {"bytes": 4 * rows * (heads + 2 * kv) * d, "flops": 3 * rows * (heads + kv) * case["rot"]}
    pairs = sum(r * n - r * (r - 1) // 2 for r, n in seqs)
    return {"bytes": 4 * rows * heads * d + 4 * keys * kv * d, "flops": 4 * pairs * heads * d}


# ---- the definition, in 64 bits -------------------------------------------------------------------------------

def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "rotary":
        return _turned_exactly(case, s["x"], s["positions"])
    if case["kind"] == "append":
        out, key, value = (s[t].double() for t in ("out", "key_pages", "value_pages"))
        for i, (rows, length) in enumerate(s["seqs"]):
            first, past = s["starts"][i], length - rows
            positions = torch.arange(past, length, device="cuda")
            q, k = (_turned_exactly(case, s[t][first:first + rows], positions) for t in ("q", "k"))
            out[first:first + rows] = q
            for page in range(past // case["page"], (length - 1) // case["page"] + 1):
                low, high = max(past, page * case["page"]), min(length, (page + 1) * case["page"])
                at = int(s["table"][i, page])
                slots, new = slice(low - page * case["page"], high - page * case["page"]), slice(low - past, high - past)
                key[at, :, slots] = k[new].permute(1, 0, 2)
                value[at, :, slots] = s["v"][first:first + rows][new].double().permute(1, 0, 2)
        return out, key, value
    out, scale = s["out"].double(), 1.5 / math.sqrt(case["d"])
    group = case["heads"] // case["kv_heads"]
    for i, (rows, length) in enumerate(s["seqs"]):
        first = s["starts"][i]
        for h in range(case["kv_heads"]):
            if case["kind"] == "paged":
                used = s["table"][i, :-(-length // case["page"])].tolist()
                key, value = (s[t][:, h][used].reshape(-1, case["d"])[:length].double()
                              for t in ("key_pages", "value_pages"))
            else:
                at = s["key_starts"][i]
                key, value = (s[t][at:at + length, h].double() for t in ("k", "v"))
            columns = torch.arange(length, device="cuda")
            for low in range(0, rows, 2048):
                high = min(rows, low + 2048)
                last = torch.arange(low, high, device="cuda") + (length - rows)
                for e in range(h * group, (h + 1) * group):
                    scores = s["q"][first + low:first + high, e].double() @ key.t() * scale
                    scores = torch.where(columns[None, :] <= last[:, None], scores, -torch.inf)
                    weights = torch.exp(scores - torch.logsumexp(scores, dim=1, keepdim=True))
                    out[first + low:first + high, e] = weights @ value
    return out


def _turned_exactly(case, x, positions):
    """x [rows, heads, d] turned as complex numbers, one pair of columns after the other."""
    rot, half = case["rot"], case["rot"] // 2
    out = x.double()
    for i in range(half):
        f = BASE ** (-2.0 * i / rot)
        magnitude = 1.0
        if case["scaling"] == "linear":
            f /= LINEAR
        elif case["scaling"] == "wavelength":
            length, w = 2 * math.pi / f, WAVELENGTH
            if length > w["original"] / w["low"]:
                f /= w["factor"]
            elif length > w["original"] / w["high"]:
                blend = (w["original"] / length - w["low"]) / (w["high"] - w["low"])
                f = (1 - blend) * f / w["factor"] + blend * f
        elif case["scaling"] == "yarn":
            y = YARN
            edge = [rot * math.log(y["original"] / (t * 2 * math.pi)) / (2 * math.log(BASE)) for t in (y["fast"], y["slow"])]
            low, high = max(math.floor(edge[0]), 0), min(math.ceil(edge[1]), rot - 1)
            ramp = min(max((i - low) / max(high - low, 0.001), 0.0), 1.0)
            f = f / y["factor"] * ramp + f * (1 - ramp)
            magnitude = 0.1 * math.log(y["factor"]) + 1.0
        angle = positions.double() * f
        turn = torch.polar(torch.full_like(angle, magnitude), angle)[:, None]
        a, b = (i, i + half) if case["layout"] == "halves" else (2 * i, 2 * i + 1)
        turned = torch.complex(x[..., a].double(), x[..., b].double()) * turn
        out[..., a], out[..., b] = turned.real, turned.imag
    return out
