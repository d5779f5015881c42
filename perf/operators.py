"""Measured cases: a student model learns from a teacher's top logits, then drafts tokens for it.

Three operators over rows of `classes` values, each through the entry points a user's program calls:

  top      opspec.top_logits     the k largest logits of each row with their indices, and the row's log normaliser
  distill  opspec.distill_ce     divergence of a student's softmax from a teacher's list of top logits, and its gradient
  verify   opspec.verify_drafts  which drafted tokens the target model accepts, and the token that follows them

With `own` false the same results come from elementary torch operations.  `exact` computes them from the
definitions in 64 bits, the gradient by automatic differentiation.
"""
from __future__ import annotations

import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "bf16": 2}


def listed():
    return [
        # one token of one sequence: the candidates that a sampler looks at
        top("top_one_row_f32", 1, 32768, 8, "f32"),
        # a teacher's pass over a batch of text: what is kept of its logits
        top("top_teacher_bf16", 4096, 131072, 64, "bf16"),
        # rows whose length is no multiple of anything, softened
        top("top_ragged_f32", 1000, 50021, 20, "f32", temperature=2.0),
        # a small classifier's batch learning from a large one's best classes
        distill("distill_small_f32", 8, 1000, 10, "f32", tail=False, temperature=4.0),
        # the wide network's batch and classes
        distill("distill_classes_f32", 8192, 1000, 16, "f32", tail=False, temperature=4.0),
        # a language model's batch of tokens, with the mass outside the teacher's list as a class of its own
        distill("distill_tokens_bf16", 4096, 131072, 64, "bf16"),
        # ragged rows, lists of different lengths, a quarter of the rows padding
        distill("distill_ragged_bf16", 777, 50021, 33, "bf16", temperature=2.0, masked=True),
        # logits kept in 32 bits, longer lists
        distill("distill_tokens_f32", 1024, 65536, 128, "f32", tail=False),
        # evaluation: the loss alone
        distill("distill_loss_bf16", 2048, 32768, 32, "bf16", backward=False),
        # one sequence being answered
        verify("verify_one_f32", 1, 4, 32768, "f32"),
        # a serving batch
        verify("verify_batch_f32", 256, 7, 131072, "f32"),
        # drafts that come from a lookup, without probabilities, of different lengths
        verify("verify_lookup_bf16", 33, 5, 50021, "bf16", lookup=True),
    ]


def top(name, rows, classes, k, dtype, temperature=1.0):
    return {"name": name, "kind": "top", "rows": rows, "classes": classes, "k": k, "dtype": dtype, "temperature": temperature}


def distill(name, rows, classes, k, dtype, tail=True, temperature=1.0, masked=False, backward=True):
    return {"name": name, "kind": "distill", "rows": rows, "classes": classes, "k": k, "dtype": dtype, "tail": tail,
            "temperature": temperature, "masked": masked, "backward": backward}


def verify(name, batch, drafts, classes, dtype, lookup=False):
    return {"name": name, "kind": "verify", "batch": batch, "drafts": drafts, "classes": classes, "dtype": dtype, "lookup": lookup}


# ------------------------------------------------------------------ drawn cases
def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind, dtype = rng.choice(["top", "distill", "distill", "verify"]), rng.choice(["f32", "bf16"])
    classes = _log(rng, 64, 200000)
    if rng.random() < 0.5:  # half of all heads have widths chosen for the hardware, half have what the data gave
        classes = (classes + 63) // 64 * 64
    if kind == "verify":
        case = verify("", _log(rng, 1, 256), rng.randint(1, 8), classes, dtype, lookup=rng.random() < 0.3)
        case["batch"] = max(1, min(case["batch"], (1 << 28) // (classes * (case["drafts"] + 1))))
    else:
        rows = max(1, min(_log(rng, 1, 16384), (1 << 28) // classes))
        k = _log(rng, 1, min(256, classes // 2))
        temperature = rng.choice([1.0, 1.0, 2.0, 4.0])
        if kind == "top":
            case = top("", rows, classes, k, dtype, temperature)
        else:
            case = distill("", rows, classes, k, dtype, rng.random() < 0.6, temperature, rng.random() < 0.3, rng.random() < 0.85)
    del case["name"]
    return case


# ------------------------------------------------------------------- the programs
def _logits(rows, classes, dtype, random):
    """Logits as a trained head gives them: a bulk, and a few classes a row that stand out."""
    x = torch.randn(rows, classes, device="cuda", generator=random).mul_(2.0)
    some = torch.randint(0, classes, (rows, 24), device="cuda", generator=random)
    x.scatter_reduce_(1, some, torch.rand(rows, 24, device="cuda", generator=random).mul_(12.0), "amax")
    return x.to(dtype)


def prepare(case, seed):
    random = torch.Generator("cuda").manual_seed(seed)
    return {"top": _prepare_top, "distill": _prepare_distill, "verify": _prepare_verify}[case["kind"]](case, random)


def _prepare_top(case, random):
    rows, k, dtype = case["rows"], case["k"], TYPES[case["dtype"]]
    return {"case": case, "logits": _logits(rows, case["classes"], dtype, random), "values": torch.empty(rows, k, dtype=dtype, device="cuda"),
            "indices": torch.empty(rows, k, dtype=torch.int64, device="cuda"), "lse": torch.empty(rows, device="cuda")}


def _prepare_distill(case, random):
    rows, classes, k, dtype = case["rows"], case["classes"], case["k"], TYPES[case["dtype"]]
    s = {"case": case, "t_lse": None, "row_weight": None, "grad": None, "loss": torch.empty(1, device="cuda"), "row_loss": torch.empty(rows, device="cuda")}
    s["logits"] = _logits(rows, classes, dtype, random)
    # a teacher that the student agrees with roughly
    teacher = torch.randn(rows, classes, device="cuda", generator=random).add_(s["logits"])
    s["t_logits"], s["t_index"] = torch.topk(teacher, k)
    s["t_logits"] = s["t_logits"].to(dtype)
    if case["tail"]:
        s["t_lse"] = torch.logsumexp(teacher / case["temperature"], 1)
    s["loss_div"] = float(rows)
    if case["masked"]:
        weight = (torch.rand(rows, device="cuda", generator=random) < 0.75).float()
        s["row_weight"] = weight
        s["loss_div"] = max(1.0, 0.75 * rows)
        keep = torch.randint(1, k + 1, (rows, 1), device="cuda", generator=random)  # lists of different lengths: -1 fills them up
        s["t_index"] = torch.where(torch.arange(k, device="cuda") < keep, s["t_index"], -1)
    if case["backward"]:
        s["grad"] = torch.empty(rows, classes, dtype=dtype, device="cuda")
    return s


def _prepare_verify(case, random):
    B, n, classes, dtype = case["batch"], case["drafts"], case["classes"], TYPES[case["dtype"]]
    draft = torch.softmax(_logits(B * n, classes, torch.float32, random), 1).to(dtype).view(B, n, classes)
    target = _logits(B * (n + 1), classes, torch.float32, random).view(B, n + 1, classes)
    target[:, :n] = draft.float().clamp_min(1e-9).log() + 0.7 * torch.randn(B, n, classes, device="cuda", generator=random)
    target = torch.softmax(target, 2).to(dtype)
    # the drafted tokens follow the draft's probabilities
    race = draft.float() / torch.empty(B, n, classes, device="cuda").exponential_(generator=random)
    s = {"case": case, "target": target, "draft": None if case["lookup"] else draft, "tokens": race.argmax(2), "lengths": None,
         "uniforms": torch.rand(B, n + 1, device="cuda", generator=random), "out": torch.empty(B, n + 1, dtype=torch.int64, device="cuda"),
         "accepted": torch.empty(B, dtype=torch.int64, device="cuda")}
    if case["lookup"]:
        s["lengths"] = torch.randint(0, n + 1, (B,), device="cuda", generator=random)
    return s


def run(state):
    if own:
        return _run_own(state)
    return {"top": _plain_top, "distill": _plain_distill, "verify": _plain_verify}[state["case"]["kind"]](state)


# ------------------------------------------------------------- the framework's calls
_dev = None


def _run_own(s):
    global _dev
    from zigrad_b200 import abi, opspec
    from zigrad_b200.device import USIZE, CudaDevice, DeviceSlice
    if _dev is None:
        _dev = CudaDevice(0, stream=torch.cuda.current_stream().cuda_stream)
    v = s.get("slices")
    if v is None:
        kinds = {torch.float32: abi.SINGLE, torch.bfloat16: abi.BF16, torch.int64: USIZE}
        v = s["slices"] = {n: DeviceSlice(t.data_ptr(), t.numel(), kinds[t.dtype]) for n, t in s.items() if isinstance(t, torch.Tensor)}
    case = s["case"]
    if case["kind"] == "top":
        _dev.dispatch(opspec.top_logits(v["logits"], case["rows"], case["classes"], case["k"], v["values"], v["indices"], lse=v["lse"],
                                        temperature=case["temperature"]))
        return {n: s[n] for n in ("values", "indices", "lse")}
    if case["kind"] == "distill":
        _dev.dispatch(opspec.distill_ce(v["logits"], v["t_index"], v["t_logits"], case["rows"], case["classes"], case["k"], v["loss"],
                                        grad=v.get("grad"), t_lse=v.get("t_lse"), row_weight=v.get("row_weight"), row_loss=v["row_loss"],
                                        temperature=case["temperature"], loss_div=s["loss_div"], accumulate=False))
        return {n: s[n] for n in ("loss", "row_loss", "grad") if s[n] is not None}
    _dev.dispatch(opspec.verify_drafts(v["target"], v["tokens"], v["uniforms"], case["batch"], case["drafts"], case["classes"], v["out"],
                                       v["accepted"], draft=v.get("draft"), lengths=v.get("lengths")))
    return {n: s[n] for n in ("out", "accepted")}


# ------------------------------------------------------------------ the plain forms
def _normaliser(z):
    m = z.amax(1, keepdim=True)
    return (m + (z - m).exp().sum(1, keepdim=True).log()).squeeze(1)


def _plain_top(s):
    x, k = s["logits"], s["case"]["k"]
    # one whole number per logit that sorts as the logit does, a lower index in front among equal ones
    bits = (x.float() + 0.0).view(torch.int32)
    bits = torch.where(bits < 0, bits ^ 0x7fffffff, bits)
    key = bits.long() * (1 << 32) + ((1 << 32) - 1 - torch.arange(x.shape[1], device="cuda"))
    key = torch.topk(key, k, dim=1).values
    indices = (1 << 32) - 1 - (key & ((1 << 32) - 1))
    return {"values": x.gather(1, indices), "indices": indices, "lse": _normaliser(x.float() / s["case"]["temperature"])}


def _plain_distill(s):
    case, T = s["case"], s["case"]["temperature"]
    z = s["logits"].float() / T
    rows, classes = z.shape
    index = s["t_index"]
    valid = (index >= 0) & (index < classes)
    index = index.clamp(0, classes - 1)
    # 64 bits for the lists and for sums over all classes: a list's mass may be near one or near zero, and a divergence is a
    # small difference of large logarithms
    u = torch.where(valid, s["t_logits"].double() / T, -math.inf)
    if case["tail"]:
        logq = u - s["t_lse"].double()[:, None]
    else:
        m = u.amax(1, keepdim=True)
        logq = u - (m + (u - m).exp().sum(1, keepdim=True).log())
    q = logq.exp()
    mass = q.sum(1)
    m = z.amax(1, keepdim=True)
    e = (z - m).exp()
    total = e.sum(1, dtype=torch.float64)
    logp = (z.gather(1, index) - m).double() - total.log()[:, None]
    row = torch.where(q > 0, q * (logq - logp), 0.0).sum(1)
    weight = s["row_weight"] if s["row_weight"] is not None else torch.ones(rows, device="cuda")
    if case["tail"]:
        rest = (1 - mass).clamp_min(0.0)
        listed_ = torch.zeros(rows, classes, dtype=torch.bool, device="cuda").scatter_(1, torch.where(valid, index, index[:, :1]), True)
        outside = e.masked_fill(listed_, 0.0)
        p_rest = outside.sum(1, dtype=torch.float64) / total
        row = row + torch.where(rest > 0, rest * (rest.log() - p_rest.log()), 0.0)
    row = (row * weight).float()
    out = {"loss": (row.double().sum() / s["loss_div"]).float().reshape(1), "row_loss": row}
    if case["backward"]:
        scale = (weight / (T * s["loss_div"]))[:, None]
        if case["tail"]:
            g = e * ((mass + rest) / total).float()[:, None] - outside * (rest / p_rest / total).float()[:, None]
        else:
            g = e * (mass / total).float()[:, None]
        g = g.scatter_add(1, index, -q.float())
        out["grad"] = (g * scale).to(s["logits"].dtype)
    return out


def _plain_verify(s):
    target, draft, tokens, u = s["target"], s["draft"], s["tokens"], s["uniforms"].double()
    B, n = tokens.shape
    at = tokens.unsqueeze(2)
    p = target[:, :n].gather(2, at).squeeze(2).double()
    q = draft.gather(2, at).squeeze(2).double() if draft is not None else torch.ones_like(p)
    lengths = s["lengths"] if s["lengths"] is not None else torch.full((B,), n, device="cuda")
    place = torch.arange(n + 1, device="cuda")
    ok = (u[:, :n] * q < p) & (place[:n] < lengths[:, None])
    accepted = ok.long().cumprod(1).sum(1)
    b = torch.arange(B, device="cuda")
    full = target[b, accepted].double()  # 64 bits: a running sum over all classes, compared with a random number
    here = accepted.clamp_max(n - 1)
    if draft is not None:
        rest = (full - draft[b, here].double()).clamp_min(0.0)
    else:
        rest = full.scatter(1, tokens[b, here][:, None], 0.0)
    w = torch.where((accepted < lengths)[:, None], rest, full)
    sums = w.cumsum(1)
    w = torch.where(sums[:, -1:] > 0, w, full)
    sums = w.cumsum(1)
    classes = w.shape[1]
    last = classes - 1 - (w > 0).flip(1).long().argmax(1)  # where rounding leaves nothing above the random share
    chosen = torch.minimum((sums <= u[:, n:] * sums[:, -1:]).sum(1), last)
    filled = torch.cat([tokens, tokens[:, :1]], 1)
    out = torch.where(place < accepted[:, None], filled, torch.where(place == accepted[:, None], chosen[:, None], -1))
    return {"out": out, "accepted": accepted}


# --------------------------------------------------------------- from the definitions
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "top":
        x = s["logits"]
        parts = [torch.sort(x[r:r + 1024].double(), dim=1, descending=True, stable=True) for r in range(0, len(x), 1024)]
        k = case["k"]
        values = torch.cat([p.values[:, :k] for p in parts])
        lse = torch.cat([torch.logsumexp(p.values / case["temperature"], 1) for p in parts])
        return {"values": values, "indices": torch.cat([p.indices[:, :k] for p in parts]), "lse": lse}
    if case["kind"] == "distill":
        parts = [_exact_distill(s, r, min(r + 512, case["rows"])) for r in range(0, case["rows"], 512)]
        out = {"loss": torch.stack([p[0] for p in parts]).sum().reshape(1), "row_loss": torch.cat([p[1] for p in parts])}
        if case["backward"]:
            out["grad"] = torch.cat([p[2] for p in parts])
        return out
    B, n = case["batch"], case["drafts"]
    out, accepted = torch.full((B, n + 1), -1, dtype=torch.int64), torch.zeros(B, dtype=torch.int64)
    tokens, u = s["tokens"].cpu(), s["uniforms"].double().cpu()
    p_at = s["target"][:, :n].double().gather(2, s["tokens"][:, :, None])[:, :, 0].cpu()
    q_at = s["draft"].double().gather(2, s["tokens"][:, :, None])[:, :, 0].cpu() if s["draft"] is not None else torch.ones(B, n).double()
    lengths = s["lengths"].cpu() if s["lengths"] is not None else torch.full((B,), n)
    for b in range(B):
        a, length = 0, int(lengths[b])
        while a < length and u[b, a] * q_at[b, a] < p_at[b, a]:
            out[b, a] = tokens[b, a]
            a += 1
        w = s["target"][b, a].double()
        if a < length:
            w = w.clone()
            if s["draft"] is not None:
                w = torch.relu(w - s["draft"][b, a].double())
            else:
                w[tokens[b, a]] = 0.0
            if float(w.sum()) == 0.0:
                w = s["target"][b, a].double()
        sums = torch.cumsum(w, 0)
        j = int(torch.searchsorted(sums, u[b, n].to(sums.device) * sums[-1], right=True))
        out[b, a] = min(j, int(w.nonzero()[-1]))
        accepted[b] = a
    return {"out": out.cuda(), "accepted": accepted.cuda()}


def _exact_distill(s, r0, r1):
    """Rows r0 .. r1: the divergence over a dense table of the teacher's mass, differentiated automatically."""
    case, T = s["case"], s["case"]["temperature"]
    x = s["logits"][r0:r1].double().requires_grad_(case["backward"])
    rows, classes = x.shape
    index, weight = s["t_index"][r0:r1], None if s["row_weight"] is None else s["row_weight"][r0:r1].double()
    there = (index >= 0) & (index < classes)
    u = (s["t_logits"][r0:r1].double() / T).masked_fill(~there, -math.inf)
    level = s["t_lse"][r0:r1].double() if case["tail"] else torch.logsumexp(u, 1)
    entries = (u - level[:, None]).exp()
    q = torch.zeros(rows, classes + 1, dtype=torch.float64, device="cuda")
    q.scatter_add_(1, torch.where(there, index, classes), torch.where(there, entries, 0.0))
    is_listed = torch.zeros(rows, classes + 1, dtype=torch.bool, device="cuda").scatter_(1, torch.where(there, index, classes), True)[:, :classes]
    q = q[:, :classes]
    logp = torch.log_softmax(x / T, 1)
    row = (torch.xlogy(q, q) - q * logp).sum(1)
    if case["tail"]:
        rest = (1.0 - q.sum(1)).clamp_min(0.0)
        log_rest = torch.logsumexp(logp.masked_fill(is_listed, -math.inf), 1)
        row = row + torch.xlogy(rest, rest) - rest * log_rest
    if weight is not None:
        row = row * weight
    loss = row.sum() / s["loss_div"]
    grad = torch.autograd.grad(loss, x)[0] if case["backward"] else None
    return loss.detach(), row.detach(), grad


# --------------------------------------------------------------------------- work
def work(case):
    """Each input read once and each output written once."""
    es = SIZES[case["dtype"]]
    if case["kind"] == "verify":
        # the drafted tokens' probabilities, and the rows that the token behind the accepted ones is sampled from
        B, n, C = case["batch"], case["drafts"], case["classes"]
        rows = 1 if case["lookup"] else 2
        return {"bytes": B * (rows * C * es + n * (8 + rows * es) + 4 * (n + 1) + 8 * (n + 2)), "flops": B * C * (rows + 1)}
    rows, C, k = case["rows"], case["classes"], case["k"]
    if case["kind"] == "top":
        return {"bytes": rows * (C * es + k * (es + 8) + 4), "flops": 4 * rows * C}
    passes = 2 if case["backward"] else 1
    lists = k * (8 + es) + 4 + (4 if case["tail"] else 0) + (4 if case["masked"] else 0)
    return {"bytes": rows * (passes * C * es + lists), "flops": rows * C * (8 if case["backward"] else 4)}
