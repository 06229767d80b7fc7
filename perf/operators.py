"""The operators of a serving step over a paged cache, as they are measured: `attention_paged`, `kv_append_paged` and
`qk_norm_rope`, each in a plain form (elementary torch operations, f32 inside, angles in f64, one rounding at the end) and
as calls of the library (`own`).

A case names sizes; the lengths of its sequences follow from `spread` (a number of its own for each case), so that the work
of a case is known without its inputs.  A batch is `seqs` sequences: sequence s brings n_s new tokens, packed one after the
other in q, k and v, and has len_s keys in the cache once they are appended.  `chunk` replaces the first sequence's number
of new tokens (a prompt's chunk beside decoding sequences), `idle` sequences at the end have one token and no key (the
empty places of a decode batch of a fixed size), `pad` tokens lie behind the last sequence and belong to none.
"""
import math
import random

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"f16": 2, "bf16": 2, "f32": 4}


def listed():
    a = dict(op="attention", nh=32, nkvh=8, dh=128, page=16, idle=0, pad=0, chunk=0, mask=1)
    c = dict(op="append", nkvh=8, dh=128, page=16, idle=0, pad=0, chunk=0, theta=10000.0)
    n = dict(op="norm", nh=32, nkvh=8, dh=128, theta=10000.0, weight="same")
    return [
        # one user's decode step in the middle of a conversation: the smallest call, where latency counts
        dict(a, name="attention decode 1", dtype="f16", seqs=1, new_min=1, new_max=1, cached_min=2047, cached_max=2047, spread=1),
        # a server's decode step: sequences from just begun to long, three places of the batch empty
        dict(a, name="attention decode 47", dtype="bf16", seqs=47, idle=3, new_min=1, new_max=1, cached_min=30, cached_max=16000, spread=2),
        # several prompts of unlike lengths at once, nothing cached, as many kv heads as query heads
        dict(a, name="attention prompts", dtype="f16", nkvh=32, page=32, seqs=7, pad=5, new_min=100, new_max=1500, cached_min=0, cached_max=0, spread=3),
        # a chunk of a long prompt: few rows for the machine, many keys for each
        dict(a, name="attention chunk of long", dtype="bf16", page=64, seqs=1, new_min=511, new_max=511, cached_min=32000, cached_max=32000, spread=4),
        # decode steps and one prompt's chunk in one launch, eight query heads to a kv head, dh 64
        dict(a, name="attention mixed", dtype="f16", nkvh=4, dh=64, page=24, seqs=25, chunk=333, new_min=1, new_max=1, cached_min=200, cached_max=7000, spread=5),
        # the longest prompt in one call: the largest case
        dict(a, name="attention prompt 8192", dtype="bf16", page=256, seqs=1, new_min=8192, new_max=8192, cached_min=0, cached_max=0, spread=6),
        # the append of one decode step of one user
        dict(c, name="append decode 1", dtype="f16", seqs=1, new_min=1, new_max=1, cached_min=2047, cached_max=2047, spread=7),
        # ... of a server's decode step, with empty places
        dict(c, name="append decode 47", dtype="bf16", seqs=47, idle=3, new_min=1, new_max=1, cached_min=30, cached_max=16000, spread=8),
        # ... of prompts
        dict(c, name="append prompts", dtype="bf16", nkvh=32, page=32, seqs=7, pad=5, new_min=700, new_max=2000, cached_min=0, cached_max=300, spread=9),
        # the norms and rotation of one token's heads
        dict(n, name="norm 1", dtype="f16", tokens=1, far=2047),
        # ... of a decode batch, far positions
        dict(n, name="norm 47", dtype="bf16", tokens=47, far=130000, theta=500000.0, weight="f32"),
        # ... of a prompt
        dict(n, name="norm prompt", dtype="bf16", tokens=8191, far=8191),
    ]


def _log_uniform(r, lo, hi):
    return lo if lo >= hi else max(lo, min(hi, int(round(math.exp(r.uniform(math.log(lo + 1), math.log(hi + 1)))) - 1)))


def _lengths(case):
    """[(new tokens, keys in the cache after they are appended)] of the case's sequences."""
    r = random.Random(case["spread"])
    out = []
    for s in range(case["seqs"]):
        n = case["chunk"] if s == 0 and case["chunk"] else _log_uniform(r, case["new_min"], case["new_max"])
        out.append((n, n + _log_uniform(r, case["cached_min"], case["cached_max"])))
    return out + [(1, 0)] * case["idle"]


def _pairs(lens, causal):
    """(query token, key) pairs that the mask keeps."""
    return sum(sum(max(0, l - n + i + 1) for i in range(n)) if causal else n * l for n, l in lens)


LARGEST = 4.0 * 128 * 32 * (8192 * 8193 / 2)  # operations of the largest listed case


def draw(rng):
    kind = rng.random()
    dh, page = rng.choice([64, 128]), rng.choice([1, 8, 16, 24, 32, 64, 100, 256])
    nkvh = rng.choice([1, 2, 4, 8, 12, 32])
    group = rng.choice([1, 2, 3, 4, 7, 8, 16])
    while nkvh * group > 64:
        group = rng.choice([1, 2])
    case = dict(dtype=rng.choice(["f16", "bf16"]), nkvh=nkvh, dh=dh)
    if kind < 0.2:
        return dict(case, op="norm", nh=nkvh * group, tokens=_log_uniform(rng, 1, 8191), far=_log_uniform(rng, 10, 1000000), dtype=rng.choice(["f16", "bf16", "f32"]),
                    theta=rng.choice([10000.0, 500000.0]), weight=rng.choice(["same", "f32"]))
    case.update(page=page, seqs=_log_uniform(rng, 1, 100), idle=rng.choice([0, 0, 1, 5]), pad=rng.choice([0, 0, 3, 17]), chunk=0, spread=rng.randrange(1 << 20))
    form = rng.choice(["decode", "decode", "prompts", "mixed", "chunks"])
    if form in ("prompts", "chunks"):
        case["seqs"] = _log_uniform(rng, 1, 12)
    case.update(new_min=1, new_max=1, cached_min=_log_uniform(rng, 1, 1000), cached_max=_log_uniform(rng, 1000, 20000))
    if form == "prompts":
        case.update(new_min=_log_uniform(rng, 1, 500), new_max=_log_uniform(rng, 500, 4000), cached_min=0, cached_max=0)
    if form == "chunks":
        case.update(new_min=_log_uniform(rng, 2, 60), new_max=_log_uniform(rng, 60, 1000))
    if form == "mixed":
        case.update(chunk=_log_uniform(rng, 16, 600))
    if kind < 0.4:
        return dict(case, op="append", theta=rng.choice([0.0, 10000.0, 500000.0]), dtype=rng.choice(["f16", "bf16", "f32"]))
    case.update(op="attention", nh=nkvh * group, mask=rng.choice([1, 1, 1, 0]))
    while True:  # smaller until it costs no more than the largest listed case, in the plain form's padded scores too
        lens = _lengths(case)
        keys = len(lens) * max(l for _, l in lens)
        if 4.0 * dh * case["nh"] * _pairs(lens, case["mask"]) <= LARGEST and keys * max(n for n, _ in lens) * case["nh"] <= 2.2e9 and keys * nkvh * dh <= 1e9:
            return case
        if case["seqs"] > 1:
            case["seqs"] = (case["seqs"] + 1) // 2
        else:
            case["new_max"] = max(case["new_min"], case["new_max"] // 2)
            case["cached_max"] = max(case["cached_min"], case["cached_max"] // 2)
            case["chunk"] //= 2


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, to=dtype):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(to)

    s = {"case": case, "dh": case["dh"]}
    if case["op"] == "norm":
        t, nh, nkvh, dh = case["tokens"], case["nh"], case["nkvh"], case["dh"]
        w = dtype if case["weight"] == "same" else torch.float32
        qkv = normal(t, (nh + 2 * nkvh) * dh, scale=1.5)  # what one projection leaves: q, k and v of a token side by side
        s.update(q=qkv[:, : nh * dh].view(t, nh, dh), k=qkv[:, nh * dh : (nh + nkvh) * dh].view(t, nkvh, dh),
                 qw=normal(dh, scale=0.2, to=torch.float32).add(1).to(w), kw=normal(dh, scale=0.2, to=torch.float32).add(1).to(w),
                 pos=torch.randint(0, case["far"] + 1, (t,), generator=g, device="cuda", dtype=torch.int32),
                 qy=torch.empty(t, nh, dh, device="cuda", dtype=dtype), ky=torch.empty(t, nkvh, dh, device="cuda", dtype=dtype))
        return s
    lens = _lengths(case)
    page, nkvh, dh = case["page"], case["nkvh"], case["dh"]
    starts = [0]
    for n, _ in lens:
        starts.append(starts[-1] + n)
    t, most = starts[-1] + case["pad"], max(l for _, l in lens)
    cols = max(1, -(-most // page))
    pages = sum(-(-l // page) for _, l in lens) + 3
    # each sequence's pages lie anywhere in the cache; entries behind its last page hold what is left there
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    used = torch.tensor([-(-l // page) for _, l in lens], device="cuda")
    first = torch.cumsum(used, 0) - used
    col = torch.arange(cols, device="cuda")
    table = order[torch.minimum(first[:, None] + col[None, :], torch.tensor(pages - 1, device="cuda"))]
    table = torch.where(col[None, :] < used[:, None], table, torch.full_like(table, -1)).contiguous()
    s.update(table=table, q_start=torch.tensor(starts, device="cuda", dtype=torch.int32), kv_len=torch.tensor([l for _, l in lens], device="cuda", dtype=torch.int32),
             most_new=max(n for n, _ in lens), most_keys=most, page=page,
             k_cache=normal(pages, nkvh, page, dh), v_cache=normal(pages, nkvh, page, dh))
    if case["op"] == "append":
        kv = normal(t, 2 * nkvh * dh)
        s.update(k=kv[:, : nkvh * dh].view(t, nkvh, dh), v=kv[:, nkvh * dh :].view(t, nkvh, dh), theta=case["theta"])
        seq = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), s["q_start"].diff().long())
        pos = torch.arange(starts[-1], device="cuda") - s["q_start"][seq] + (s["kv_len"] - s["q_start"].diff())[seq]
        s["pos"] = torch.cat([pos.clamp(min=0), torch.zeros(case["pad"], device="cuda", dtype=pos.dtype)]).to(torch.int32)
    else:
        nh = case["nh"]
        s.update(q=normal(t, nh, dh, scale=1.5), o=torch.full((t, nh, dh), 0.125, device="cuda", dtype=dtype), mask=case["mask"], scale=1.0 / math.sqrt(dh))
    return s


# ---- the plain forms

def _rotate(x, pos, theta):
    """[a, b] <- [a cos - b sin, a sin + b cos] for the adjacent pairs (2 k, 2 k + 1) of x [t, heads, dh] (f32), angle pos * theta^(-2 k / dh)."""
    half = x.shape[-1] // 2
    freq = theta ** (-torch.arange(half, device=x.device, dtype=torch.float64) / half)
    ang = pos.double()[:, None, None] * freq
    c, s = ang.cos().float(), ang.sin().float()
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)


def _norm(s):
    def one(x, w):
        x = x.float()
        return _rotate(x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w.float(), s["pos"], s["case"]["theta"]).to(s["q"].dtype)
    return {"q": one(s["q"], s["qw"]), "k": one(s["k"], s["kw"])}


def _tokens(s, t):
    """Of every token of the batch: its sequence, its number there, whether it belongs to one at all."""
    tok = torch.arange(t, device=s["q_start"].device)
    start = s["q_start"].long()
    seq = (torch.searchsorted(start, tok, right=True) - 1).clamp(max=len(start) - 2)
    return seq, tok - start[seq], tok < start[-1]


def _append(s):
    k, v = s["k"], s["v"]
    seq, i, real = _tokens(s, k.shape[0])
    new = s["q_start"].diff().long()
    key = s["kv_len"].long()[seq] - new[seq] + i
    real = real & (key >= 0)
    if s["theta"]:
        k = _rotate(k.float(), s["pos"], s["theta"]).to(k.dtype)
    # tokens without a place write token 0's values to token 0's place once more
    key = torch.where(real, key, key[0])
    seq = torch.where(real, seq, seq[0])
    at, row = s["table"][seq, key // s["page"]].long(), key % s["page"]
    s["k_cache"][at, :, row] = torch.where(real[:, None, None], k, k[0])
    s["v_cache"][at, :, row] = torch.where(real[:, None, None], v, v[0])
    return {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _attention(s):
    q, dh = s["q"], s["dh"]
    t, nh, nkvh = q.shape[0], q.shape[1], s["k_cache"].shape[1]
    start, length = s["q_start"].long(), s["kv_len"].long()
    ns, n, most = len(length), s["most_new"], s["most_keys"]
    j = torch.arange(most, device=q.device)
    at = s["table"][:, j // s["page"]].long().clamp(min=0)
    kept = (j < length[:, None])[:, :, None, None]
    k = torch.where(kept, s["k_cache"][at, :, j % s["page"]], 0).float()  # [seqs, keys, kv heads, dh]
    v = torch.where(kept, s["v_cache"][at, :, j % s["page"]], 0).float()
    i = torch.arange(n, device=q.device)
    rows = (start[:-1, None] + i).clamp(max=t - 1)
    x = q[rows].float().view(ns, n, nkvh, nh // nkvh, dh).permute(0, 2, 3, 1, 4).reshape(ns * nkvh, -1, dh)
    p = torch.bmm(x, k.permute(0, 2, 3, 1).reshape(ns * nkvh, dh, most).contiguous()).view(ns, nh, n, most).mul_(s["scale"])
    limit = (length - start.diff())[:, None] + i + 1 if s["mask"] else length[:, None].expand(ns, n)
    keep = (j < torch.minimum(limit, length[:, None])[:, :, None])[:, None]
    p.masked_fill_(~keep, -math.inf)
    top = p.amax(-1, keepdim=True).clamp(min=-1e30)
    p = p.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    y = torch.bmm(p.view(ns * nkvh, -1, most), v.permute(0, 2, 1, 3).reshape(ns * nkvh, most, dh).contiguous()).view(ns, nh, n, dh)
    y = torch.where(total > 0, y / total, 0)
    seq, i, real = _tokens(s, t)
    y = y.permute(0, 2, 1, 3)[seq, i.clamp(max=n - 1)].to(q.dtype)
    s["o"].copy_(torch.where(real[:, None, None], y, s["o"]))
    return s["o"]


# ---- the library's calls

_library = {}


def _ophip():
    """The library, its device, a torch stream's queue and the operators: what a program makes once."""
    if not _library:
        import os
        import sys
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "operators-rs_amd"))
        import ophip
        gpu = ophip.Gpu(torch.cuda.current_device())
        _library.update(ophip=ophip, gpu=gpu, queues={}, attention=ophip.AttentionPaged(gpu), append=ophip.KvAppendPaged(gpu), norm=ophip.QkNormRope(gpu))
    return _library


def _queue():
    """The library's view of torch's current stream."""
    lib, handle = _library, torch.cuda.current_stream().cuda_stream
    if handle not in lib["queues"]:
        lib["queues"][handle] = lib["ophip"].ExternalStream(lib["gpu"], handle)
    return lib["queues"][handle]


def _layout(x, dims=None):
    """(layout, address) of a torch tensor, its dimensions in the order `dims`."""
    dt = _library["ophip"].dt
    codes = {torch.float16: dt.F16, torch.bfloat16: dt.BF16, torch.float32: dt.F32, torch.int32: dt.U32, torch.int64: dt.U64}
    dims = range(x.dim()) if dims is None else dims
    return _library["ophip"].TensorLayout(codes[x.dtype], [x.shape[d] for d in dims], [x.stride(d) * x.element_size() for d in dims]), x.data_ptr()


def _bind(s):
    """The call's arguments and workspace: they name buffers and sizes, so a serving loop keeps them beside its buffers."""
    lib, op = _ophip(), s["case"]["op"]
    ophip = lib["ophip"]
    if op == "norm":
        args = ophip.QkNormRopeArgs(*_layout(s["qy"]), *_layout(s["q"]), *_layout(s["qw"]), *_layout(s["ky"]), *_layout(s["k"]), *_layout(s["kw"]), *_layout(s["pos"]),
                                    1e-6, s["case"]["theta"])
        out = {"q": s["qy"], "k": s["ky"]}
    else:
        cache = _layout(s["k_cache"]) + _layout(s["v_cache"])
        batch = _layout(s["table"]) + _layout(s["q_start"]) + _layout(s["kv_len"])
        if op == "append":
            args = ophip.KvAppendPagedArgs(*_layout(s["k"], (1, 0, 2)), *_layout(s["v"], (1, 0, 2)), *_layout(s["pos"]), *cache, *batch, s["theta"])
            out = {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}
        else:
            args = ophip.AttentionPagedArgs(*_layout(s["q"], (1, 0, 2)), *cache, *_layout(s["o"], (1, 0, 2)), *batch, s["mask"], s["scale"])
            out = s["o"]
    need = lib[op].scheme(args, 1 << 40)
    space = torch.empty(need, dtype=torch.uint8, device="cuda") if need else None
    return lib[op], args, space, (space.data_ptr(), need) if need else None, out


def run(s):
    if own:
        if "call" not in s:
            s["call"] = _bind(s)
        op, args, _, workspace, out = s["call"]
        op.launch(args, workspace, _queue())
        return out
    return {"norm": _norm, "append": _append, "attention": _attention}[s["case"]["op"]](s)


# ---- what a pass cannot do without

def work(case):
    e, dh, nkvh = BYTES[case["dtype"]], case["dh"], case["nkvh"]
    if case["op"] == "norm":
        values = case["tokens"] * (case["nh"] + nkvh) * dh
        return {"bytes": 2 * values * e + 4 * case["tokens"], "flops": 7 * values}
    lens = _lengths(case)
    meta = 4 * (2 * len(lens) + 1 + sum(-(-l // case["page"]) for _, l in lens))
    if case["op"] == "append":
        values = sum(n for n, l in lens if l) * nkvh * dh
        return {"bytes": 4 * values * e + meta, "flops": (3 if case["theta"] else 1) * values}
    nh = case["nh"]
    return {"bytes": e * (2 * nh * dh * sum(n for n, _ in lens) + 2 * nkvh * dh * sum(l for _, l in lens)) + meta, "flops": 4 * dh * nh * _pairs(lens, case["mask"])}


# ---- the definitions in 64 bits

def _turn(x, pos, theta):
    """x [t, heads, dh] (f64) as complex numbers, each multiplied by exp(i pos theta^(-k / half))."""
    t, heads, dh = x.shape
    z = torch.view_as_complex(x.reshape(t, heads, dh // 2, 2).contiguous())
    w = torch.exp(-math.log(theta) * torch.arange(dh // 2, dtype=torch.float64, device=x.device) * 2.0 / dh)
    ang = pos.to(torch.float64).view(t, 1, 1) * w
    return torch.view_as_real(z * torch.polar(torch.ones_like(ang), ang)).reshape(t, heads, dh)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        out = {}
        for name, w in (("q", s["qw"]), ("k", s["kw"])):
            x = s[name].double()
            x = x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + 1e-6).sqrt() * w.double()
            out[name] = _turn(x, s["pos"], case["theta"])
        return out
    lens, page = _lengths(case), case["page"]
    table, at = s["table"].cpu(), 0
    if case["op"] == "append":
        kc, vc = s["k_cache"].double(), s["v_cache"].double()
        k = _turn(s["k"].double(), s["pos"], case["theta"]) if case["theta"] else s["k"].double()
        for r, (n, l) in enumerate(lens):
            for i in range(max(0, n - l), n):
                slot = l - n + i
                p = int(table[r, slot // page])
                kc[p, :, slot % page], vc[p, :, slot % page] = k[at + i], s["v"][at + i].double()
            at += n
        return {"k_cache": kc, "v_cache": vc}
    o, group = s["o"].double(), case["nh"] // case["nkvh"]
    for r, (n, l) in enumerate(lens):
        o[at : at + n] = 0
        if l:
            ids = table[r, : -(-l // page)].long().cuda()
            for h in range(case["nkvh"]):
                k = s["k_cache"][ids, h].reshape(-1, s["dh"])[:l].double()
                v = s["v_cache"][ids, h].reshape(-1, s["dh"])[:l].double()
                for x in range(h * group, (h + 1) * group):
                    z = s["q"][at : at + n, x].double() @ k.T.contiguous() * s["scale"]
                    if case["mask"]:
                        z = z + torch.full_like(z, -math.inf).triu(l - n + 1)
                    if l >= n or not case["mask"]:
                        o[at : at + n, x] = torch.softmax(z, -1) @ v
        at += n
    return o
