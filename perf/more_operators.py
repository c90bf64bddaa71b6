"""Operators of models that keep a state per sequence, and of the beam search that moves these states, as cases that can be timed and compared.

A batch of rows names its sequences through seq_info, int32 [4][n_seq]: a sequence's first row, its count of rows (tokens), its state slot, and 1 where it
begins (its state and its last inputs then count as zeros).

Kinds of case:

  conv     short causal convolution over the tokens of every channel, a bias, silu; the last inputs of a sequence wait in its slot
  scan     selective state space scan: d = softplus(dt + bias), h[c][n] <- exp(d a[c][n]) h[c][n] + d x b[n], y = sum_n c[n] h[c][n] + skip x, times silu(z)
  select   the best successors of a request's beams: score of the beam + logit - log(sum of exp(logits)), over all beams and tokens; ties go to the lowest index
  reorder  slots become what other slots held before, all at once, in all layers
"""
import ctypes as C
import math
import random

import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
DEV = "cuda"


def listed():
    return [
        # the next token of 64 chats goes through the convolution in front of the scan
        {"name": "conv_step", "kind": "conv", "type": "f32", "seqs": 64, "new_lo": 1, "new_hi": 1, "channels": 4096, "taps": 4, "bias": True, "begin": 0.0},
        # prompts that arrive together, some of them continuations
        {"name": "conv_prompts", "kind": "conv", "type": "bf16", "seqs": 5, "new_lo": 131, "new_hi": 2001, "channels": 8192, "taps": 4, "bias": True, "begin": 0.6},
        # one user's next token: latency is what counts
        {"name": "scan_one_token", "kind": "scan", "type": "f32", "seqs": 1, "new_lo": 1, "new_hi": 1, "channels": 2048, "d_state": 16, "groups": 1, "gate": True, "skip": True, "begin": 0.0},
        # 96 chats decode together: their states go through the device once
        {"name": "scan_batch", "kind": "scan", "type": "bf16", "seqs": 96, "new_lo": 1, "new_hi": 1, "channels": 8192, "d_state": 16, "groups": 1, "gate": True, "skip": True, "begin": 0.0},
        # one long prompt of a small model: few channels, so the tokens have to be shared out
        {"name": "scan_prompt", "kind": "scan", "type": "f32", "seqs": 1, "new_lo": 4096, "new_hi": 4096, "channels": 2048, "d_state": 16, "groups": 1, "gate": False, "skip": True, "begin": 1.0},
        # ragged prompts that arrive together, some of them continuations
        {"name": "scan_prompts_ragged", "kind": "scan", "type": "bf16", "seqs": 6, "new_lo": 37, "new_hi": 1501, "channels": 5120, "d_state": 16, "groups": 1, "gate": True, "skip": True, "begin": 0.5},
        # a wide state, channels in groups that have b and c of their own, a width that is no power of two
        {"name": "scan_wide_state", "kind": "scan", "type": "f16", "seqs": 2, "new_lo": 701, "new_hi": 999, "channels": 2600, "d_state": 64, "groups": 4, "gate": True, "skip": False, "begin": 0.5},
        # four full prompts of a large model
        {"name": "scan_prompts_long", "kind": "scan", "type": "bf16", "seqs": 4, "new_lo": 2048, "new_hi": 2048, "channels": 8192, "d_state": 16, "groups": 1, "gate": True, "skip": True, "begin": 1.0},
        # one request, four beams
        {"name": "select_one", "kind": "select", "type": "f32", "requests": 1, "beams": 4, "vocab": 32000, "keep": 8, "ended": 0.0, "masked": 0.0},
        # 48 requests of eight beams, a large vocabulary, tokens that a grammar forbids, beams that have ended
        {"name": "select_batch", "kind": "select", "type": "bf16", "requests": 48, "beams": 8, "vocab": 128257, "keep": 8, "ended": 0.1, "masked": 0.2},
        # the states of one request's beams, all layers of a small model
        {"name": "reorder_one", "kind": "reorder", "layers": 24, "requests": 1, "beams": 4, "slots": 9, "state": 32768, "tail": 6144},
        # 16 requests of eight beams, some layers of a large model
        {"name": "reorder_batch", "kind": "reorder", "layers": 8, "requests": 16, "beams": 8, "slots": 130, "state": 131072, "tail": 24576},
    ]


def spread_over(rng, lo, hi):
    """A whole number, spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["conv", "conv", "scan", "scan", "scan", "scan", "select", "select", "reorder"])
    t = rng.choice(["f32", "bf16", "f16"])
    if kind in ("conv", "scan"):
        channels = rng.choice([64, 1024, 1536, 2048, 2560, 4096, 5120, 8192, spread_over(rng, 33, 8192)])
        if rng.random() < 0.4:
            seqs, new = spread_over(rng, 1, 128), rng.choice([1, 1, 1, 2, 5])
        else:
            seqs, new = rng.choice([1, 1, 2, 4, 7]), spread_over(rng, 8, 4096)
        base = {"kind": kind, "type": t, "seqs": seqs, "channels": channels, "begin": rng.choice([0.0, 0.5, 1.0])}
        if kind == "conv":
            new = max(1, min(new, (1 << 26) // (seqs * channels)))
            return base | {"new_lo": max(1, new // rng.choice([1, 3, 16])), "new_hi": new, "taps": rng.choice([2, 3, 4, 4, 4, 4, 5, 8]), "bias": rng.random() < 0.8}
        n = rng.choice([16, 16, 16, 16, 8, 32, 64, 128, rng.randint(1, 128)])
        new = max(1, min(new, (1 << 29) // (seqs * channels * n)))
        groups = rng.choice([g for g in (1, 1, 1, 2, 4, 8) if channels % g == 0])
        return base | {"new_lo": max(1, new // rng.choice([1, 3, 16])), "new_hi": new, "d_state": n, "groups": groups, "gate": rng.random() < 0.7, "skip": rng.random() < 0.8}
    if kind == "select":
        beams = rng.choice([1, 2, 4, 4, 5, 8, 16, 32])
        vocab = rng.choice([32000, 32003, 50257, 128256, 151936, spread_over(rng, 50, 200000)])
        requests = max(1, min(spread_over(rng, 1, 64), (1 << 26) // (beams * vocab)))
        return {"kind": "select", "type": t, "requests": requests, "beams": beams, "vocab": vocab, "keep": rng.choice([1, beams, beams, 2 * beams]),
                "ended": rng.choice([0.0, 0.0, 0.3]), "masked": rng.choice([0.0, 0.0, 0.2, 0.9])}
    beams, state = rng.choice([2, 4, 8, 8, 16]), 4 * spread_over(rng, 64, 65536)
    requests = max(1, min(spread_over(rng, 1, 32), (1 << 25) // (beams * state)))
    layers = max(1, min(spread_over(rng, 1, 48), (1 << 27) // (requests * beams * state)))
    return {"kind": "reorder", "layers": layers, "requests": requests, "beams": beams, "slots": requests * beams + rng.choice([0, 1, 7]), "state": state,
            "tail": rng.choice([0, 3 * max(1, state // 16), spread_over(rng, 1, 20000)])}


# ------------------------------------------------------------------------------------------------ sizes that follow from a case
def between(lo, hi, n):
    """n whole numbers from lo to hi, evenly spread, in an order that goes with the numbers."""
    v = [lo + (hi - lo) * i // max(1, n - 1) if n > 1 else hi for i in range(n)]
    random.Random(n * 7919 + lo * 31 + hi).shuffle(v)
    return v


def plan_of(case):
    """New tokens and slot of every sequence, and whether it begins."""
    n = case["seqs"]
    new = between(case["new_lo"], case["new_hi"], n)
    rng = random.Random(n * 31 + case["channels"])
    return new, rng.sample(range(n + 2), n), [i < round(case["begin"] * n) for i in range(n)]


# ------------------------------------------------------------------------------------------------ inputs
def normal(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device=DEV) * std


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = {"case": case}
    if case["kind"] == "select":
        return prepare_select(case, g, s)
    if case["kind"] == "reorder":
        return prepare_reorder(case, seed, g, s)
    new, slots, begin = plan_of(case)
    tokens, ch, t = sum(new), case["channels"], TORCH[case["type"]]
    first = [sum(new[:i]) for i in range(len(new))]
    s |= {"tokens": tokens, "longest": max(new), "slots": case["seqs"] + 2, "seq_info": torch.tensor([first, new, slots, [int(b) for b in begin]], dtype=torch.int32, device=DEV)}
    s["dst"] = torch.zeros(tokens, ch, dtype=t, device=DEV)
    if case["kind"] == "conv":
        k = case["taps"]
        s |= {"x": normal(g, tokens, ch).to(t), "w": normal(g, ch, k, std=1 / math.sqrt(k)), "bias": normal(g, ch, std=0.2) if case["bias"] else None}
        s["tail"] = normal(g, s["slots"], k - 1, ch).to(t).float()
        return s
    n, x = case["d_state"], normal(g, tokens, ch)
    s["x"] = (x * torch.sigmoid(x)).to(t)
    # steps of 0.001 to 0.1 where dt is 0, as such layers begin their training; rates 1, 2, 3 ..
    step = torch.exp(math.log(0.001) + (math.log(0.1) - math.log(0.001)) * torch.rand(ch, generator=g, device=DEV))
    s["dt"], s["dt_bias"] = normal(g, tokens, ch, std=0.7).to(t), step + torch.log(-torch.expm1(-step))
    s["a"] = -(torch.arange(1, n + 1, device=DEV) * torch.exp(normal(g, ch, n, std=0.2))).contiguous()
    bc = normal(g, tokens, 2 * case["groups"] * n).to(t)  # a product's two halves
    s["b"], s["c"] = bc[:, :case["groups"] * n], bc[:, case["groups"] * n:]
    s["skip"] = 1 + normal(g, ch, std=0.1) if case["skip"] else None
    s["z"] = normal(g, tokens, ch).to(t) if case["gate"] else None
    s["state"] = normal(g, s["slots"], ch, n, std=0.3)
    return s


def prepare_select(case, g, s):
    rows, v = case["requests"] * case["beams"], case["vocab"]
    # a few tokens lead: what a trained model's rows look like
    logits = normal(g, rows, v, std=2.0)
    lead = torch.randint(0, v, (rows, min(v, 24)), generator=g, device=DEV)
    logits.scatter_add_(1, lead, 6 + normal(g, *lead.shape, std=2.0))
    if case["masked"]:
        logits.masked_fill_(torch.rand(rows, v, generator=g, device=DEV) < case["masked"], -math.inf)
    s["logits"] = logits.to(TORCH[case["type"]])
    s["score"] = -10 * torch.rand(rows, generator=g, device=DEV) - 1
    s["ended"] = (torch.rand(rows, generator=g, device=DEV) < case["ended"]).to(torch.int32)
    s["slot"] = torch.randperm(rows, generator=g, device=DEV).to(torch.int32)
    n = case["requests"] * case["keep"]
    s |= {"to_score": torch.zeros(n, device=DEV)} | {k: torch.zeros(n, dtype=torch.int32, device=DEV) for k in ("to_beam", "to_token", "to_slot")}
    return s


def moves(case, seed):
    """Slots of the beams, and the slot that each becomes: of its own request, good beams more often than others."""
    rng = random.Random(seed)
    at = rng.sample(range(case["slots"]), case["requests"] * case["beams"])
    src = []
    for r in range(case["requests"]):
        mine = at[r * case["beams"]:(r + 1) * case["beams"]]
        src += rng.choices(mine, weights=[0.6 ** i for i in range(len(mine))], k=len(mine))
    return src, at


def prepare_reorder(case, seed, g, s):
    src, dst = moves(case, seed)
    s |= {"src": torch.tensor(src, dtype=torch.int32, device=DEV), "dst": torch.tensor(dst, dtype=torch.int32, device=DEV)}
    s["states"] = [normal(g, case["slots"], n) for _ in range(case["layers"]) for n in (case["state"], case["tail"]) if n]
    return s


# ------------------------------------------------------------------------------------------------ the plain forms
def softplus(x):
    return torch.clamp(x, min=0) + torch.log1p(torch.exp(-x.abs()))


def sequence_of(seq_info, tokens):
    """Sequence and place in it of every row."""
    first, count = seq_info[0].long(), seq_info[1].long()
    seq = torch.repeat_interleave(torch.arange(count.numel(), device=DEV), count, output_size=tokens)
    return seq, torch.arange(tokens, device=DEV) - first[seq]


def plain_conv(s):
    c, info = s["case"], s["seq_info"].long()
    k, x = c["taps"], s["x"].float()
    seq, at = sequence_of(s["seq_info"], s["tokens"])
    before = torch.where(info[3].bool()[:, None, None], 0.0, s["tail"][info[2]])  # [n_seq, taps - 1, channels]
    seen = torch.cat([before.reshape(-1, c["channels"]), x])
    # where the input j places before row i of the sequence lies
    def place(row_seq, i):
        return torch.where(i < 0, row_seq * (k - 1) + i + k - 1, (k - 1) * c["seqs"] + info[0][row_seq] + i)
    back = torch.arange(k, device=DEV) - k + 1
    y = (seen[place(seq[:, None], at[:, None] + back)] * s["w"].T).sum(1)
    if s["bias"] is not None:
        y = y + s["bias"]
    s["dst"].copy_(y / (1 + torch.exp(-y)))
    s["tail"][info[2]] = seen[place(torch.arange(c["seqs"], device=DEV)[:, None], info[1][:, None] + back[1:] - 1)]
    return {"y": s["dst"], "tail": s["tail"]}


def plain_scan(s):
    """All tokens at once: h_t = decay_t h_(t-1) + add_t by doubling, the first token of a sequence taking its state in."""
    c, info = s["case"], s["seq_info"].long()
    group = torch.arange(c["channels"], device=DEV) // (c["channels"] // c["groups"])
    d = softplus(s["dt"].float() + s["dt_bias"])
    x = s["x"].float()
    b, cc = (s[k].float().reshape(s["tokens"], c["groups"], c["d_state"])[:, group] for k in ("b", "c"))
    decay = torch.exp(d[..., None] * s["a"])
    h = (d * x)[..., None] * b
    begins = info[0]
    h[begins] += torch.where(info[3].bool()[:, None, None], 0.0, decay[begins] * s["state"][info[2]])
    decay[begins] = 0
    k = 1
    while k < s["longest"]:
        h[k:] += decay[k:] * h[:-k].clone()
        decay[k:] = decay[k:] * decay[:-k]
        k *= 2
    y = (h * cc).sum(-1)
    if s["skip"] is not None:
        y = y + s["skip"] * x
    if s["z"] is not None:
        z = s["z"].float()
        y = y * z / (1 + torch.exp(-z))
    s["dst"].copy_(y)
    s["state"][info[2]] = h[begins + info[1] - 1]
    return {"y": s["dst"], "state": s["state"]}


def plain_select(s):
    """In 64 bits: scores of different beams may lie next to each other."""
    c = s["case"]
    r, beams, v, keep = c["requests"], c["beams"], c["vocab"], c["keep"]
    logits = s["logits"].float() + 0.0
    wide = logits.double()
    top = wide.amax(1, keepdim=True)
    norm = top + torch.log(torch.exp(wide - top).sum(1, keepdim=True))
    norm = torch.where(top == -math.inf, 0.0, norm)  # a row that allows nothing
    # a row's best: the logit's bits in an order of whole numbers, the place behind them
    bits = logits.view(torch.int32).long()
    key = torch.where(bits < 0, -(bits & 0x7fffffff), bits) * (1 << 31) + (v - 1 - torch.arange(v, device=DEV))
    best = torch.topk(key, min(keep, v), dim=1).indices  # [rows, n]
    score = s["score"].double()[:, None] + (torch.gather(wide, 1, best) - norm)
    # an ended beam has one successor, itself
    ended, lead = s["ended"].bool()[:, None], torch.arange(best.shape[1], device=DEV) == 0
    score = torch.where(ended, torch.where(lead, s["score"].double()[:, None], -math.inf), score)
    best = torch.where(ended, 0, best)
    flat = (torch.arange(beams, device=DEV).repeat(r)[:, None] * v + best).reshape(r, -1)
    order = torch.argsort(flat, dim=1, stable=True)
    flat, score = torch.gather(flat, 1, order), torch.gather(score.reshape(r, -1), 1, order)
    order = torch.argsort(score, dim=1, descending=True, stable=True)[:, :keep]
    flat, score = torch.gather(flat, 1, order), torch.gather(score, 1, order)
    there = score > -math.inf
    beam = torch.div(flat, v, rounding_mode="floor")
    slot = torch.gather(s["slot"].reshape(r, beams).long(), 1, beam)
    n = flat.shape[1]
    s["to_score"].reshape(r, keep).fill_(-math.inf)[:, :n] = score
    for name, what in (("to_beam", beam), ("to_token", flat % v), ("to_slot", slot)):
        s[name].reshape(r, keep).fill_(-1)[:, :n] = torch.where(there, what, -1)
    return {"score": s["to_score"], "beam": s["to_beam"], "token": s["to_token"], "slot": s["to_slot"]}


def plain_reorder(s):
    src, dst = s["src"].long(), s["dst"].long()
    for x in s["states"]:
        x[dst] = x[src]
    return s["states"]


def run(s):
    kind = s["case"]["kind"]
    if own:
        return run_own(s, kind)
    return {"conv": plain_conv, "scan": plain_scan, "select": plain_select, "reorder": plain_reorder}[kind](s)


# ------------------------------------------------------------------------------------------------ the framework's calls
def plan(s):
    """The argument structures of a state's call, made once, as a program keeps them."""
    from koboldcpp_b200 import lib as L
    c, ll = s["case"], L.lib()

    def at(name):
        return s[name].data_ptr() if s.get(name) is not None else None

    kind = {"f32": L.F32, "f16": L.F16, "bf16": L.BF16}[c.get("type", "f32")]
    if c["kind"] == "conv":
        a = L.SsmConvArgs(x=at("x"), x_stride=c["channels"], w=at("w"), bias=at("bias"), seq_info=at("seq_info"), tail=at("tail"), slot_stride=(c["taps"] - 1) * c["channels"],
                          dst=at("dst"), dst_stride=c["channels"], n_seq=c["seqs"], n_slots=s["slots"], n_tokens=s["tokens"], max_new=s["longest"], channels=c["channels"],
                          taps=c["taps"], silu=1, type=kind)
        ref = C.byref(a)
        return a, lambda: L.check(ll.b200_op_ssm_conv(ref, None)), {"y": s["dst"], "tail": s["tail"]}
    if c["kind"] == "scan":
        bc = 2 * c["groups"] * c["d_state"]
        a = L.SsmScanArgs(x=at("x"), x_stride=c["channels"], dt=at("dt"), dt_stride=c["channels"], b=at("b"), b_stride=bc, c=at("c"), c_stride=bc, z=at("z"), z_stride=c["channels"],
                          a=at("a"), dt_bias=at("dt_bias"), d=at("skip"), seq_info=at("seq_info"), state=at("state"), slot_stride=c["channels"] * c["d_state"], dst=at("dst"),
                          dst_stride=c["channels"], n_seq=c["seqs"], n_slots=s["slots"], n_tokens=s["tokens"], max_new=s["longest"], channels=c["channels"], d_state=c["d_state"],
                          groups=c["groups"], softplus=1, type=kind)
        ref, n = C.byref(a), ll.b200_ssm_scan_workspace_bytes(C.byref(a))
        room = torch.empty(max(16, n), dtype=torch.uint8, device=DEV)
        return a, lambda: L.check(ll.b200_op_ssm_scan(ref, room.data_ptr(), n, None)), {"y": s["dst"], "state": s["state"]}
    if c["kind"] == "select":
        a = L.BeamSelectArgs(logits=at("logits"), logits_stride=c["vocab"], score=at("score"), ended=at("ended"), slot=at("slot"), to_score=at("to_score"), to_beam=at("to_beam"),
                             to_token=at("to_token"), to_slot=at("to_slot"), n_requests=c["requests"], n_beams=c["beams"], n_vocab=c["vocab"], n_keep=c["keep"], end_token=0, type=kind)
        ref, n = C.byref(a), ll.b200_beam_select_workspace_bytes(C.byref(a))
        room = torch.empty(max(16, n), dtype=torch.uint8, device=DEV)
        return a, lambda: L.check(ll.b200_op_beam_select(ref, room.data_ptr(), n, None)), {"score": s["to_score"], "beam": s["to_beam"], "token": s["to_token"], "slot": s["to_slot"]}
    a = (L.SlotState * len(s["states"]))(*[L.SlotState(x.data_ptr(), 4 * x.shape[1], 4 * x.shape[1]) for x in s["states"]])
    src, dst, m = s["src"].data_ptr(), s["dst"].data_ptr(), s["src"].numel()
    return a, lambda: L.check(ll.b200_op_state_reorder(a, len(a), src, dst, m, c["slots"], None, None)), s["states"]


def run_own(s, kind):
    if "plan" not in s:
        s["plan"] = plan(s)
    _, call, outputs = s["plan"]
    call()
    return outputs


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    if c["kind"] == "select":
        rows = c["requests"] * c["beams"]
        return {"bytes": rows * c["vocab"] * SIZE[c["type"]] + 12 * rows + 16 * c["requests"] * c["keep"], "flops": 4 * rows * c["vocab"]}
    if c["kind"] == "reorder":
        # of a request's beams that are drawn by their weights, so many are some other's successor, and so many have a successor on another slot
        w = [0.6 ** i for i in range(c["beams"])]
        p = [x / sum(w) for x in w]
        read = sum(1 - (1 - q) ** (c["beams"] - 1) for q in p)
        moved = c["beams"] - sum(p)
        return {"bytes": int(4 * c["layers"] * c["requests"] * (c["state"] + c["tail"]) * (read + moved)), "flops": 0}
    new, _, begin = plan_of(c)
    tokens, ch, es, n_old = sum(new), c["channels"], SIZE[c["type"]], c["seqs"] - sum(begin)
    if c["kind"] == "conv":
        k = c["taps"]
        return {"bytes": 2 * tokens * ch * es + 4 * ch * (k + c["bias"]) + 4 * ch * (k - 1) * (c["seqs"] + n_old), "flops": tokens * ch * (2 * k + 5)}
    n = c["d_state"]
    rows = (3 + c["gate"]) * ch + 2 * c["groups"] * n
    return {"bytes": tokens * rows * es + 4 * ch * (n + 1 + c["skip"]) + 4 * ch * n * (c["seqs"] + n_old), "flops": tokens * ch * (7 * n + 8 + 2 * c["skip"] + 5 * c["gate"])}


# ------------------------------------------------------------------------------------------------ the definition, in 64 bits
def conv64(s):
    c, y, tail = s["case"], [], s["tail"].double()
    for first, count, slot, begins in s["seq_info"].T.tolist():
        old = torch.zeros_like(tail[slot]) if begins else tail[slot]
        u = torch.cat([old, s["x"][first:first + count].double()])
        o = sum(u[j:j + count] * s["w"][:, j].double() for j in range(c["taps"]))
        o = o + (s["bias"].double() if s["bias"] is not None else 0)
        y.append(o * torch.sigmoid(o))
        tail[slot] = u[count:]
    return {"y": torch.cat(y), "tail": tail}


def scan64(s):
    """Token by token; sequences side by side, those that have ended stay as they are."""
    c, info = s["case"], s["seq_info"].long()
    of = torch.arange(c["channels"], device=DEV) // (c["channels"] // c["groups"])
    x, d = s["x"].double(), torch.nn.functional.softplus(s["dt"].double() + s["dt_bias"].double())
    b, cc = (s[k].double().reshape(s["tokens"], c["groups"], c["d_state"]) for k in ("b", "c"))
    h = s["state"].double()[info[2]] * (1 - info[3])[:, None, None]
    y, a = torch.zeros_like(x), s["a"].double()
    counts = info[1].tolist()
    for i in range(s["longest"]):
        live = torch.tensor([j for j, m in enumerate(counts) if m > i], device=DEV)
        t = info[0][live] + i
        now = torch.exp(d[t][..., None] * a) * h[live] + (d[t] * x[t])[..., None] * b[t][:, of]
        y[t] = (now * cc[t][:, of]).sum(-1)
        h[live] = now
    if s["skip"] is not None:
        y += s["skip"].double() * x
    if s["z"] is not None:
        y *= torch.nn.functional.silu(s["z"].double())
    state = s["state"].double()
    state[info[2]] = h
    return {"y": y, "state": state}


def select64(s):
    c, best = s["case"], []
    for r in range(c["requests"]):
        rows = slice(r * c["beams"], (r + 1) * c["beams"])
        p = torch.log_softmax(s["logits"][rows].double(), dim=1) + s["score"][rows].double()[:, None]
        p[s["ended"][rows].bool() | torch.isnan(p[:, 0])] = -math.inf  # (a row that allows nothing has no logarithm)
        p[:, 0] = torch.where(s["ended"][rows].bool(), s["score"][rows].double(), p[:, 0])
        p = torch.cat([p.reshape(-1), torch.full((c["keep"],), -math.inf, device=DEV, dtype=torch.float64)])
        best.append(torch.sort(p, descending=True).values[:c["keep"]])
    return {"score": torch.cat(best), "beam": None, "token": None, "slot": None}


def exact(case, seed):
    if case["kind"] == "reorder":
        return None  # copies
    return {"conv": conv64, "scan": scan64, "select": select64}[case["kind"]](prepare(case, seed))
