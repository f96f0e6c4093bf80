"""What the operators on the frames' logits of packed lines cost: the cases that are measured.

A recognizer's head gives every frame of a line one logit a class.  Four operators work on the
frames of many lines, end to end in one array, line i's rows [line_at[i], line_at[i + 1]):

  adapters    the head's 1x1 projection with each line's own low-rank adapter beside it
  rules       a line's rules on its frames' logits: penalties for characters it had already, a
              bias, a set of allowed classes
  greedy      greedy CTC decoding of the lines under their rules
  candidates  the k likeliest classes but the blank of each frame under its line's rules

`own` false computes their plain forms in elementary torch operations, `own` true calls the
library.  Class 0 is the CTC blank.
"""
from __future__ import annotations

import math

import torch

own = False

BLANK = 0
SETS, BIASES = 8, 4  # allowed-class sets and bias tables a program keeps for its fields and languages


# ------------------------------------------------------------------------------------ the cases

def listed():
    return [
        # one line of the crop rule's test box (62 frames): what a single correction costs
        dict(name="adapters_line", op="adapters", frames=62, lines=1, tail=0, k=256, classes=800, adapters=8, rank=8, half=False),
        # a page of 64 lines, a few customers' adapters among them
        dict(name="adapters_page", op="adapters", frames=4800, lines=64, tail=16, k=256, classes=800, adapters=16, rank=16, half=False),
        # a device run's head product, [65536, 256] x [256, 800], some 75 frames a line
        dict(name="adapters_run", op="adapters", frames=65536, lines=870, tail=0, k=256, classes=800, adapters=32, rank=16, half=False),
        # the 12,000-class head (192 channels), float16 logits
        dict(name="adapters_cjk", op="adapters", frames=4096, lines=64, tail=0, k=192, classes=12000, adapters=8, rank=32, half=True),
        # lines of one frame, each with an adapter of its own choice
        dict(name="adapters_rows", op="adapters", frames=512, lines=512, tail=0, k=256, classes=800, adapters=64, rank=16, half=False),
        # the rows of a beam's step: 64 hypotheses, each with what it has read so far
        dict(name="rules_rows", op="rules", frames=64, lines=64, tail=0, classes=800, history=40, half=False),
        # a device run's logits
        dict(name="rules_run", op="rules", frames=65536, lines=870, tail=64, classes=800, history=64, half=False),
        # hypotheses over the 12,000 classes, float16
        dict(name="rules_cjk", op="rules", frames=4099, lines=1025, tail=0, classes=12000, history=200, half=True),
        # a page of 64 lines
        dict(name="greedy_page", op="greedy", frames=4800, lines=64, tail=0, classes=800, history=64, half=False),
        # a device run
        dict(name="greedy_run", op="greedy", frames=65536, lines=870, tail=0, classes=800, history=64, half=False),
        # the unsure lines of a page
        dict(name="candidates_page", op="candidates", frames=1201, lines=16, tail=0, classes=800, history=64, topk=10, half=False),
        # many lines over the 12,000 classes, float16, the largest k
        dict(name="candidates_cjk", op="candidates", frames=4096, lines=55, tail=0, classes=12000, history=64, topk=16, half=True),
    ]


MOST = 65536 * 800  # frames x classes of the largest listed case


def draw(rng):
    def spread(lo, hi):  # whole numbers, spread over their logarithm
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))

    op = rng.choice(["adapters", "rules", "greedy", "candidates"])
    classes = spread(2, 12000)
    frames = spread(1, min(65536, MOST // classes))
    # lines from one frame each to the whole width of a page
    lines = frames if rng.random() < 0.2 else max(1, frames // spread(1, 512))
    c = dict(op=op, frames=frames, lines=lines, tail=rng.choice([0, 0, spread(1, 200)]), classes=classes, half=rng.random() < 0.4)
    if op == "adapters":
        c["k"] = 8 * rng.randint(2, 40)
        c["adapters"] = spread(1, 64)
        c["rank"] = rng.randint(1, 1024 // c["adapters"] if c["adapters"] > 16 else 64)
        return c
    c["history"] = rng.choice([0, spread(1, 300)])
    if op == "candidates":
        c["topk"] = rng.randint(1, min(16, classes - 1))
    return c


def words_of(classes):
    return (classes + 31) // 32


# ------------------------------------------------------------------------------------ what a program has in hand

def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    frames, lines, classes = case["frames"], case["lines"], case["classes"]
    rows, half = frames + case["tail"], case["half"]
    kind = torch.float16 if half else torch.float32

    def rand(*size):
        return torch.rand(*size, generator=g, device=dev)

    def randn(*size):
        return torch.randn(*size, generator=g, device=dev)

    def whole(lo, hi, *size):
        return torch.randint(lo, hi, size, generator=g, device=dev, dtype=torch.int32)

    s = dict(case=dict(case), rows=rows)
    if lines == frames:
        at = torch.arange(lines + 1, device=dev, dtype=torch.int32)
    else:
        share = torch.cumsum(0.4 + rand(lines).double(), 0)
        at = torch.zeros(lines + 1, device=dev, dtype=torch.int32)
        at[1:] = torch.round(share / share[-1] * frames).int()
    s["line_at"] = at
    if case["op"] == "adapters":
        k, n, r = case["k"], case["adapters"], case["rank"]
        # the distributions of the reference's head test: features N(0, 1), weights N(0, 0.06), biases N(0, 0.5)
        s["x"] = randn(rows, k).half()
        s["w"] = (randn(classes, k) * 0.06).half()
        s["b"] = randn(classes) * 0.5
        s["down"] = (randn(n, r, k) / math.sqrt(k)).half()
        s["up"] = (randn(n, classes, r) * 0.1).half()
        s["scale"] = 0.5 + rand(n)
        s["adapter"] = whole(-1, n, lines)  # -1: the head alone
        s["logits"] = torch.zeros(rows, classes, device=dev, dtype=kind)
        if own:
            s["plan"] = head_of(s)
        return s
    # a trained head's frames: four in five blank, a character's frames side by side
    z = randn(rows, classes) * 2.0
    z[:, BLANK] += torch.where(rand(rows) < 0.8, 7.0, 0.0)
    said = whole(0, classes, rows // 3 + 1).long().repeat_interleave(3)[:rows]
    z.scatter_add_(1, said[:, None], 6.0 * rand(rows, 1))
    s["logits"] = z.to(kind)
    del z
    had = whole(0, case["history"] + 1, lines)
    s["history_at"] = torch.zeros(lines + 1, device=dev, dtype=torch.int32)
    s["history_at"][1:] = torch.cumsum(had, 0).int()
    s["history"] = (classes * rand(max(1, lines * case["history"])) ** 3).int().clamp_(max=classes - 1)  # few characters, often
    s["repeat"] = 1.0 + 0.5 * rand(lines)
    s["presence"] = 0.5 * rand(lines)
    s["frequency"] = 0.2 * rand(lines)
    s["bias"] = 0.5 * randn(BIASES, classes)
    s["bias_of"] = whole(-1, BIASES, lines)
    keep = rand(SETS, words_of(classes) * 32) < torch.linspace(0.02, 1.0, SETS, device=dev)[:, None]
    keep[:, BLANK] = True
    keep[2] = False  # a field whose grammar leaves nothing
    bit = torch.ones(32, device=dev, dtype=torch.int64) << torch.arange(32, device=dev)
    packed = (keep.view(SETS, -1, 32) * bit).sum(2)
    s["allowed"] = torch.where(packed >= 1 << 31, packed - (1 << 32), packed).int()
    s["set_of"] = whole(-1, SETS, lines)
    if case["op"] == "rules":
        s["out"] = torch.zeros(rows, classes, device=dev, dtype=kind)
    elif case["op"] == "greedy":
        s["counts"] = torch.zeros(lines, device=dev, dtype=torch.int32)
        s["ids"] = torch.zeros(rows, device=dev, dtype=torch.int32)
        s["starts"] = torch.zeros(rows, device=dev, dtype=torch.int32)
        s["probs"] = torch.zeros(rows, device=dev)
    else:
        s["ids"] = torch.zeros(rows, case["topk"], device=dev, dtype=torch.int32)
        s["logp"] = torch.zeros(rows, case["topk"], device=dev)
        s["blank"] = torch.zeros(rows, device=dev)
    if own:
        s["plan"] = lines_of(s)
    return s


def package():
    import os
    import sys
    at = os.path.join(os.getcwd(), "carbon-ocr_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    from carbon_rec import native
    return native


def head_of(s):
    """The head's file, opened once with its adapters."""
    import struct
    native = package()
    classes, k = s["w"].shape
    file = b"CTCHEAD1" + struct.pack("<ii", classes, k) + s["w"].cpu().numpy().tobytes() + s["b"].cpu().numpy().tobytes()
    sets = zip(s["down"].cpu().numpy(), s["up"].cpu().numpy(), s["scale"].tolist())
    return native.Adapters(native.ctc_head_blob(file), list(sets))


def lines_of(s):
    """The descriptors of the lines' logits and of their rules."""
    native = package()
    case = s["case"]
    kind = native.FP16 if case["half"] else native.FP32
    frames = native.LineLogits(s["logits"].data_ptr(), kind, case["classes"], case["classes"], s["rows"], case["lines"], s["line_at"].data_ptr())
    p = {f: s[f].data_ptr() for f in ("history", "history_at", "repeat", "presence", "frequency", "bias", "bias_of", "allowed", "set_of")}
    return frames, native.Rules(biases=BIASES, sets=SETS, **p)


# ------------------------------------------------------------------------------------ one pass

def run(s):
    return run_own(s) if own else PLAIN[s["case"]["op"]](s)


def run_own(s):
    native = package()
    case, stream = s["case"], torch.cuda.current_stream().cuda_stream
    if case["op"] == "adapters":
        s["plan"].logits(s["x"].data_ptr(), s["rows"], case["lines"], s["line_at"].data_ptr(), s["adapter"].data_ptr(),
                         s["logits"].data_ptr(), native.FP16 if case["half"] else native.FP32, stream=stream)
        return s["logits"]
    frames, rules = s["plan"]
    if case["op"] == "rules":
        native.logit_rules(frames, rules, s["out"].data_ptr(), native.FP16 if case["half"] else native.FP32, stream=stream)
        return s["out"]
    if case["op"] == "greedy":
        native.ctc_greedy_lines(frames, rules, s["counts"].data_ptr(), s["ids"].data_ptr(), s["starts"].data_ptr(),
                                s["probs"].data_ptr(), stream=stream)
        return dict(counts=s["counts"], ids=s["ids"], starts=s["starts"], probs=s["probs"])
    native.candidates_lines(frames, rules, case["topk"], s["ids"].data_ptr(), s["logp"].data_ptr(), s["blank"].data_ptr(),
                            stream=stream)
    return dict(ids=s["ids"], logp=s["logp"], blank=s["blank"])


def line_of_rows(s):
    """Each frame's line."""
    at, frames = s["line_at"], s["case"]["frames"]
    row = torch.arange(frames, device=at.device, dtype=torch.int32)
    return torch.searchsorted(at, row, right=True) - 1


def plain_adapters(s):
    frames = s["case"]["frames"]
    n, r, k = s["down"].shape
    which = s["adapter"].long()[line_of_rows(s)]
    x = s["x"][:frames].float()
    z = x @ s["w"].float().t() + s["b"]
    # every adapter's down product, all but the frame's own set to 0, then every up product at once
    h = (x @ s["down"].float().view(n * r, k).t()).view(frames, n, r)
    h = h * (torch.where(which[:, None] == torch.arange(n, device=x.device), s["scale"], 0.0))[:, :, None]
    z = z + h.view(frames, n * r) @ s["up"].float().transpose(1, 2).reshape(n * r, -1)
    s["logits"][:frames] = z.to(s["logits"].dtype)
    return s["logits"]


def plain_ruled(s):
    """The frames' logits under their lines' rules, 32 bits, each operation rounded on its own."""
    case = s["case"]
    frames, lines, classes = case["frames"], case["lines"], case["classes"]
    line = line_of_rows(s)
    z = s["logits"][:frames].float()
    # how often each line had each class
    entry = torch.arange(s["history"].numel(), device=z.device, dtype=torch.int32)
    of = torch.searchsorted(s["history_at"], entry, right=True) - 1
    real = of < lines
    cell = torch.where(real, of * classes + s["history"], lines * classes)
    count = torch.zeros(lines * classes + 1, device=z.device).index_add_(0, cell, real.float())[:-1].view(lines, classes)
    less = count * s["frequency"][:, None] + s["presence"][:, None]
    had, rep = (count > 0)[line], s["repeat"][line][:, None]
    z = torch.where(had, torch.where(z > 0, z / rep, z * rep) - less[line], z)
    # the bias table
    table = s["bias_of"].long()
    add = torch.where((table >= 0)[:, None], s["bias"][table.clamp(min=0)], 0.0)
    z = z + add[line]
    # the allowed classes
    bits = (s["allowed"][:, :, None] >> torch.arange(32, device=z.device)) & 1
    keep = bits.reshape(SETS, -1)[:, :classes] != 0
    field = s["set_of"].long()
    keep = (field < 0)[:, None] | keep[field.clamp(min=0)]
    return torch.where(keep[line], z, -math.inf)


def plain_rules(s):
    s["out"][:s["case"]["frames"]] = plain_ruled(s).to(s["out"].dtype)
    return s["out"]


def lowest_of(hit, width):
    """The first true place of each row (0 where there is none)."""
    place = torch.arange(width, device=hit.device, dtype=torch.int32)
    first = torch.where(hit, place, width).amin(1)
    return torch.where(first == width, 0, first)


def plain_greedy(s):
    case = s["case"]
    frames, lines = case["frames"], case["lines"]
    line, z = line_of_rows(s), plain_ruled(s)
    best = z.amax(1)
    some = best > -math.inf
    arg = torch.where(some, lowest_of(z == best[:, None], case["classes"]), BLANK)
    total = torch.exp(z - torch.where(some, best, 0.0)[:, None]).sum(1)
    prob = torch.where(some, 1.0 / total, 0.0)
    # a character begins where a frame's class is not the blank and not the frame's before it in the line
    before = torch.cat([arg.new_full((1,), -1), arg[:-1]])
    row = torch.arange(frames, device=z.device)
    start = s["line_at"].long()[line]
    begins = (arg != BLANK) & ((arg != before) | (row == start))
    nth = torch.cumsum(begins, 0)  # characters up to and with this frame, of all lines
    upto = torch.cat([nth.new_zeros(1), nth])[s["line_at"].long()]
    s["counts"].copy_((upto[1:] - upto[:-1]).int())
    place = start + nth - 1 - upto[:-1][line]  # where the frame's character goes
    spare = torch.full_like(place, frames)
    ids = torch.full((frames + 1,), -1, device=z.device, dtype=torch.int32).scatter_(0, torch.where(begins, place, spare), arg.int())
    starts = torch.full((frames + 1,), -1, device=z.device, dtype=torch.int32).scatter_(0, torch.where(begins, place, spare), (row - start).int())
    probs = torch.zeros(frames + 1, device=z.device).scatter_reduce_(0, torch.where(arg != BLANK, place, spare), prob, "amax")
    s["ids"][:frames], s["starts"][:frames], s["probs"][:frames] = ids[:-1], starts[:-1], probs[:-1]
    return dict(counts=s["counts"], ids=s["ids"], starts=s["starts"], probs=s["probs"])


def plain_candidates(s):
    case = s["case"]
    frames, k = case["frames"], case["topk"]
    z = plain_ruled(s)
    best = z.amax(1, keepdim=True)
    some = best > -math.inf
    base = torch.where(some, best, 0.0)
    total = torch.log(torch.where(some, torch.exp(z - base).sum(1, keepdim=True), 1.0))
    top, at = torch.sort(z[:, 1:], dim=1, descending=True, stable=True)
    top, at = top[:, :k], at[:, :k] + 1
    s["ids"][:frames] = torch.where(top > -math.inf, at, -1).int()
    s["logp"][:frames] = (top - base) - total
    s["blank"][:frames] = ((z[:, :1] - base) - total)[:, 0]
    return dict(ids=s["ids"], logp=s["logp"], blank=s["blank"])


PLAIN = dict(adapters=plain_adapters, rules=plain_rules, greedy=plain_greedy, candidates=plain_candidates)


# ------------------------------------------------------------------------------------ what a pass cannot do without

def work(case):
    f, c, lines, size = case["frames"], case["classes"], case["lines"], 2 if case["half"] else 4
    if case["op"] == "adapters":
        k, n, r = case["k"], case["adapters"], case["rank"]
        moved = 2 * f * k + 2 * c * k + 4 * c + n * (2 * r * (k + c) + 4) + 8 * lines + f * c * size
        return {"bytes": moved, "flops": 2 * f * (k * c + r * (k + c))}
    # the logits once; the lines' places, their rules and what the rules name
    moved = f * c * size + lines * (4 + 4 + 12 + 8 + 2 * case["history"]) + BIASES * c * 4 + SETS * words_of(c) * 4
    if case["op"] == "rules":
        return {"bytes": moved + f * c * size, "flops": 4 * f * c}
    if case["op"] == "greedy":
        return {"bytes": moved + 4 * lines + 12 * f, "flops": 7 * f * c}
    return {"bytes": moved + f * (8 * case["topk"] + 4), "flops": 8 * f * c}


# ------------------------------------------------------------------------------------ the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    at = s["line_at"].tolist()
    if case["op"] == "adapters":
        out, frames = s["logits"].double(), case["frames"]
        x = s["x"][:frames].double()
        out[:frames] = torch.addmm(s["b"].double(), x, s["w"].double().T)
        of = [a for i, a in enumerate(s["adapter"].tolist()) for _ in range(at[i], at[i + 1])]  # each frame's
        of = torch.tensor(of, device=x.device)
        for a in range(case["adapters"]):
            mine = torch.nonzero(of == a)[:, 0]
            delta = (x[mine] @ s["down"][a].double().T) @ s["up"][a].double().T
            out.index_add_(0, mine, s["scale"][a].double() * delta)
        return out
    double = case["op"] == "rules"
    ruled = exact_rules(s, at, torch.float64 if double else torch.float32)
    if double:
        out = s["out"].double()
        out[:case["frames"]] = ruled
        return out
    return (exact_greedy if case["op"] == "greedy" else exact_candidates)(s, at, ruled.double())


def exact_rules(s, at, kind):
    """Line by line.  The decoders' logits are 32-bit numbers by definition, each step rounded."""
    case = s["case"]
    classes = case["classes"]
    z = s["logits"][:case["frames"]].to(kind)
    had_at, table, field = s["history_at"].tolist(), s["bias_of"].tolist(), s["set_of"].tolist()
    words = s["allowed"].long() & 0xFFFFFFFF
    place = torch.arange(classes, device=z.device)
    allowed = torch.bitwise_and(words[:, place // 32] >> (place % 32), 1).bool()
    for i in range(case["lines"]):
        rows = z[at[i]:at[i + 1]]
        if rows.shape[0] == 0:
            continue
        had = s["history"][had_at[i]:had_at[i + 1]].long()
        if had.numel():
            seen, times = torch.unique(had, return_counts=True)
            v = rows[:, seen]
            rep = s["repeat"][i:i + 1].to(kind)
            v = torch.where(v > 0, torch.div(v, rep), torch.mul(v, rep))
            rows[:, seen] = v - (times.to(kind) * s["frequency"][i].to(kind) + s["presence"][i].to(kind))
        if table[i] >= 0:
            rows += s["bias"][table[i]].to(kind)
        if field[i] >= 0:
            rows.masked_fill_(~allowed[field[i]], -math.inf)
    return z


def exact_greedy(s, at, z):
    case = s["case"]
    counts, ids, starts, probs = (s[f].tolist() for f in ("counts", "ids", "starts", "probs"))
    top = z.amax(1)
    first = torch.where(z == top[:, None], torch.arange(case["classes"], device=z.device), case["classes"]).amin(1)
    first, none = first.tolist(), torch.isneginf(top).tolist()
    like = torch.exp(top - torch.logsumexp(z, 1)).tolist()
    for i in range(case["lines"]):
        n, prev = at[i], BLANK
        for t in range(at[i], at[i + 1]):
            ids[t], starts[t], probs[t] = -1, -1, 0.0
            c = BLANK if none[t] else first[t]
            if c != BLANK and c != prev:
                ids[n], starts[n], probs[n] = c, t - at[i], like[t]
                n += 1
            elif c != BLANK:
                probs[n - 1] = max(probs[n - 1], like[t])
            prev = c
        counts[i] = n - at[i]
    whole = dict(dtype=torch.int32, device=z.device)
    return dict(counts=torch.tensor(counts, **whole), ids=torch.tensor(ids, **whole), starts=torch.tensor(starts, **whole),
                probs=torch.tensor(probs, dtype=torch.float64, device=z.device))


def exact_candidates(s, at, z):
    case = s["case"]
    k, frames = case["topk"], case["frames"]
    p = torch.log_softmax(z, 1)
    p = torch.where(torch.isnan(p), -math.inf, p)  # frames whose rules leave nothing
    ids, logp, blank = s["ids"].clone(), s["logp"].double(), s["blank"].double()
    blank[:frames] = p[:, 0]
    z = z.clone()
    z[:, BLANK] = -math.inf
    place = torch.arange(case["classes"], device=z.device)
    for q in range(k):  # the lowest class of the highest logit, then without it
        top = z.amax(1, keepdim=True)
        c = torch.where(z == top, place, case["classes"]).amin(1)
        gone = torch.isneginf(top[:, 0])
        ids[:frames, q] = torch.where(gone, -1, c).int()
        logp[:frames, q] = torch.where(gone, -math.inf, p.gather(1, c[:, None])[:, 0])
        z.scatter_(1, c[:, None], -math.inf)
    return dict(ids=ids, logp=logp, blank=blank)
