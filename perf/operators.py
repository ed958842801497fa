"""The operators of a decoder block over packed tokens, as cases that can be timed and compared.

Four operators, each reached through ``tacker_b200.ops``:

  attention   softmax(scale * Q K^T) V over sequences of different lengths packed in one array, causal or not, with fewer
              key/value heads than query heads; prompts, chunks of a prompt behind a cache, and single tokens
  rope        the split of a fused projection's product into q, k and v heads with rotary positions on q and k, the new
              keys and values written to their rows of a cache
  norm        y = x + s * g * norm(a) and h = norm(y) in one pass: the norms behind and before a block, its gate and the
              scale of its residual branch
  i8          rows rounded to 8-bit integers with a scale each, and their product with a matrix of 8-bit integers with a
              scale for each output channel

``run`` computes them from elementary torch operations, or with the framework's kernels where ``own`` is true.
"""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"f32": 0, "f16": 1, "bf16": 2}
WORKSPACE_BYTES = 64 << 20


# ---- the cases -----------------------------------------------------------------------------------------------------
def listed():
    return [
        # one short prompt with the head layout of this repository's BERT task: what a call costs when there is little to do
        dict(name="attention_short_prompt", op="attention", type="f16", heads=12, kv_heads=12, dim=64, causal=True,
             seqs=1, q_lo=128, q_hi=128, past_lo=0, past_hi=0, slab=0, len_seed=1),
        # the prompts of one serving step, packed: sixteen of very different lengths, grouped heads
        dict(name="attention_packed_prompts", op="attention", type="bf16", heads=32, kv_heads=8, dim=128, causal=True,
             seqs=16, q_lo=1, q_hi=1111, past_lo=0, past_hi=0, slab=0, len_seed=2),
        # one long prompt: the tensor cores' share of the work
        dict(name="attention_long_prompt", op="attention", type="f16", heads=16, kv_heads=4, dim=128, causal=True,
             seqs=1, q_lo=8192, q_hi=8192, past_lo=0, past_hi=0, slab=0, len_seed=3),
        # one decoding step of a batch: a token for each sequence, caches of all lengths in slabs of one size
        dict(name="attention_token_batch", op="attention", type="bf16", heads=32, kv_heads=8, dim=128, causal=True,
             seqs=64, q_lo=1, q_hi=1, past_lo=0, past_hi=4095, slab=4096, len_seed=4),
        # one decoding step of two long conversations: few rows, a long axis
        dict(name="attention_token_long", op="attention", type="f16", heads=16, kv_heads=2, dim=128, causal=True,
             seqs=2, q_lo=1, q_hi=1, past_lo=60001, past_hi=65535, slab=65536, len_seed=5),
        # a packed prompt's projections: 32 query and 8 key/value heads out of one fp32 product with its bias
        dict(name="rope_prompt", op="rope", x_type="f32", out_type="bf16", tokens=8191, heads=32, kv_heads=8, dim=128,
             rot=128, interleaved=False, bias=True, first=0, base=10000.0, factor=1.0, magnitude=1.0, slots=0),
        # a decoding step far into a long context: half of each head turned, pairs side by side, keys into a cache
        dict(name="rope_tokens", op="rope", x_type="f16", out_type="f16", tokens=61, heads=16, kv_heads=2, dim=128,
             rot=64, interleaved=True, bias=False, first=1000000, base=500000.0, factor=8.0, magnitude=1.2, slots=4096),
        # the residual stream of a packed prompt between two blocks
        dict(name="norm_prompt", op="norm", kind="rms", a_type="bf16", x_type="bf16", h_type="bf16", rows=8191, cols=4096,
             post=True, pre=True, gate_rows=0, scale=1.0, eps=1e-6),
        # a few rows of this repository's BERT width with a gate for each sequence: latency
        dict(name="norm_rows", op="norm", kind="layer", a_type="f32", x_type="f32", h_type="f16", rows=37, cols=768,
             post=False, pre=True, gate_rows=16, scale=0.5, eps=1e-5),
        # a decoding step's projection: a few rows, the weights' bytes
        dict(name="i8_tokens", op="i8", x_type="bf16", out_type="bf16", rows=16, outs=8192, cols=4096, bias=False),
        # odd rows and outputs with a bias
        dict(name="i8_ragged", op="i8", x_type="f16", out_type="f32", rows=1001, outs=1234, cols=1040, bias=True),
        # a packed prompt's projection
        dict(name="i8_prompt", op="i8", x_type="bf16", out_type="bf16", rows=8192, outs=8192, cols=4096, bias=False),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(("attention", "attention", "attention", "rope", "norm", "i8"))
    if op == "attention":
        group = rng.choice((1, 1, 2, 3, 4, 5, 7, 8, 16))
        kv_heads = rng.choice((1, 2, 3, 4, 8))
        while group * kv_heads > 32:
            kv_heads = max(1, kv_heads // 2)
        c = dict(op=op, type=rng.choice(("f16", "bf16")), heads=group * kv_heads, kv_heads=kv_heads,
                 dim=rng.choice((64, 64, 80, 96, 128, 128)), causal=rng.random() < 0.8, len_seed=rng.randrange(1 << 30))
        kind = rng.choice(("prompt", "token", "chunk"))
        if kind == "prompt":
            hi = _log(rng, 2, 6000)
            c.update(seqs=_log(rng, 1, 40), q_lo=rng.choice((1, max(1, hi // 2))), q_hi=hi, past_lo=0, past_hi=0, slab=0)
        elif kind == "token":
            past = _log(rng, 1, 40000)
            c.update(seqs=_log(rng, 1, 128), q_lo=1, q_hi=1, past_lo=rng.choice((0, past // 2)), past_hi=past,
                     slab=past + 1 + rng.randrange(64))
        else:
            past, hi = _log(rng, 1, 8000), _log(rng, 2, 600)
            c.update(seqs=_log(rng, 1, 16), q_lo=rng.choice((1, max(1, hi // 2))), q_hi=hi, past_lo=0, past_hi=past,
                     slab=past + hi + rng.randrange(64))
        # no more scores and no larger a cache than the listed cases have
        longest = c["q_hi"] + c["past_hi"]
        c["seqs"] = max(1, min(c["seqs"], 800_000_000 // (c["q_hi"] * longest * c["heads"]),
                               260_000_000 // (longest * kv_heads * c["dim"])))
        return c
    if op == "rope":
        dim = rng.choice((64, 80, 96, 128))
        kv_heads = rng.choice((1, 2, 4, 8))
        tokens = _log(rng, 1, 6000)
        return dict(op=op, x_type=rng.choice(("f32", "f16", "bf16")), out_type=rng.choice(("f16", "bf16")), tokens=tokens,
                    heads=kv_heads * rng.choice((1, 3, 4)), kv_heads=kv_heads, dim=dim,
                    rot=rng.choice((dim, dim, dim // 2, dim // 4 // 2 * 2)), interleaved=rng.random() < 0.5,
                    bias=rng.random() < 0.5, first=rng.choice((0, _log(rng, 1, 2_000_000))),
                    base=rng.choice((10000.0, 500000.0, 1000000.0)), factor=rng.choice((1.0, 4.0, 32.0)),
                    magnitude=rng.choice((1.0, 1.1, 1.35)), slots=rng.choice((0, tokens + 100)))
    if op == "norm":
        rows, cols = _log(rng, 1, 8000), rng.choice((_log(rng, 8, 8192), 128 * rng.randint(1, 64)))
        rows = max(1, min(rows, 33_000_000 // cols))
        return dict(op=op, kind=rng.choice(("rms", "layer")), a_type=rng.choice(("f32", "f16", "bf16")),
                    x_type=rng.choice(("f32", "f16", "bf16")), h_type=rng.choice(("f32", "f16", "bf16")), rows=rows,
                    cols=cols, post=rng.random() < 0.6, pre=rng.random() < 0.8, gate_rows=rng.choice((-1, 0, 1, 7, 128)),
                    scale=rng.choice((1.0, 0.5, 0.22)), eps=rng.choice((1e-6, 1e-5)))
    rows, outs, cols = _log(rng, 1, 8000), _log(rng, 8, 8192), 16 * _log(rng, 1, 512)
    while rows * outs * cols > 8192 * 8192 * 4096:
        rows = max(1, rows // 2)
    return dict(op=op, x_type=rng.choice(("f32", "f16", "bf16")), out_type=rng.choice(("f32", "f16", "bf16")), rows=rows,
                outs=outs, cols=cols, bias=rng.random() < 0.5)


def _lengths(case):
    """Query and key lengths of each sequence: the case's alone, the same for every seed."""
    rng = random.Random(case["len_seed"])
    q = [rng.randint(case["q_lo"], case["q_hi"]) for _ in range(case["seqs"])]
    return q, [n + rng.randint(case["past_lo"], case["past_hi"]) for n in q]


# ---- inputs --------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def normal(*shape, type="f32", scale=1.0):
        return (torch.randn(*shape, generator=g, device=dev, dtype=torch.float32) * scale).to(TYPES[type])

    s = dict(case=case)
    if case["op"] == "attention":
        ql, kl = _lengths(case)
        total, n = sum(ql), case["seqs"]
        starts = [case["slab"] * i for i in range(n)] if case["slab"] else [sum(kl[:i]) for i in range(n)]
        rows = case["slab"] * n if case["slab"] else sum(kl)
        ints = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
        s.update(q=normal(total, case["heads"], case["dim"], type=case["type"]),
                 k=normal(rows, case["kv_heads"], case["dim"], type=case["type"]),
                 v=normal(rows, case["kv_heads"], case["dim"], type=case["type"]),
                 q_start=ints([sum(ql[:i]) for i in range(n + 1)]), k_start=ints(starts), k_len=ints(kl), total=total,
                 rows=rows, max_q=max(ql), max_k=max(kl), scale=1.0 / math.sqrt(case["dim"]),
                 out=torch.zeros(total + 1, case["heads"], case["dim"], dtype=TYPES[case["type"]], device=dev),
                 lse=torch.zeros(total + 1, case["heads"], dtype=torch.float32, device=dev),
                 workspace=torch.empty(WORKSPACE_BYTES, dtype=torch.uint8, device=dev))
    elif case["op"] == "rope":
        t, h, hk, d = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        out = TYPES[case["out_type"]]
        rows = case["slots"] or t
        # a model's rotary plan: turns of a pair for each position, stretched for a longer context
        i = torch.arange(0, case["rot"], 2, dtype=torch.float64, device=dev)
        s.update(x=normal(t, (h + 2 * hk) * d, type=case["x_type"]),
                 bias=normal((h + 2 * hk) * d, scale=0.1) if case["bias"] else None,
                 pos=(case["first"] + torch.randperm(2 * t, generator=g, device=dev)[:t]).to(torch.int32),
                 turns=case["base"] ** (-i / max(1, case["rot"])) / (2 * math.pi * case["factor"]),
                 slots=torch.randperm(rows, generator=g, device=dev)[:t] if case["slots"] else None,
                 q=torch.zeros(t, h, d, dtype=out, device=dev), k=torch.zeros(rows, hk, d, dtype=out, device=dev),
                 v=torch.zeros(rows, hk, d, dtype=out, device=dev))
    elif case["op"] == "norm":
        r, c = case["rows"], case["cols"]
        layer = case["kind"] == "layer"
        gates = {-1: None, 0: 1}.get(case["gate_rows"], -(-r // max(1, case["gate_rows"])))
        s.update(a=normal(r, c, type=case["a_type"], scale=3.0), x=normal(r, c, type=case["x_type"], scale=2.0),
                 post_gamma=1 + normal(c, scale=0.2), post_beta=normal(c, scale=0.2) if layer else None,
                 pre_gamma=1 + normal(c, scale=0.2), pre_beta=normal(c, scale=0.2) if layer else None,
                 gate=None if gates is None else normal(gates, c), y=torch.zeros(r, c, dtype=TYPES[case["x_type"]], device=dev),
                 h=torch.zeros(r, c, dtype=TYPES[case["h_type"]], device=dev))
    else:
        m, n, k = case["rows"], case["outs"], case["cols"]
        # weights as a user keeps them: rounded once, a scale for each output channel
        w = normal(n, k, scale=1.0 / math.sqrt(k))
        ws = w.abs().amax(1).clamp_min(1e-30) / 127
        s.update(x=normal(m, k, type=case["x_type"]), w=(w / ws[:, None]).round().clamp(-127, 127).to(torch.int8), ws=ws,
                 bias=normal(n) if case["bias"] else None, codes=torch.zeros(m, k, dtype=torch.int8, device=dev),
                 scales=torch.zeros(m, dtype=torch.float32, device=dev),
                 out=torch.zeros(m, n, dtype=TYPES[case["out_type"]], device=dev))
    return s


# ---- one pass ------------------------------------------------------------------------------------------------------
def run(s):
    op = s["case"]["op"]
    if own:
        return {"attention": _own_attention, "rope": _own_rope, "norm": _own_norm, "i8": _own_i8}[op](s)
    return {"attention": _attention, "rope": _rope, "norm": _norm, "i8": _i8}[op](s)


def _attention(s):
    c, dev = s["case"], s["q"].device
    n, h, hk, d, mq, mk = c["seqs"], c["heads"], c["kv_heads"], c["dim"], s["max_q"], s["max_k"]
    qs, ks, kl = s["q_start"].long(), s["k_start"].long(), s["k_len"].long()
    ql = qs[1:] - qs[:-1]
    t, j = torch.arange(mq, device=dev), torch.arange(mk, device=dev)
    q_ok, k_ok = t < ql[:, None], j < kl[:, None]
    qi = torch.where(q_ok, qs[:-1, None] + t, s["total"])
    kj = torch.where(k_ok, ks[:, None] + j, 0)
    q = s["q"].float()[qi.clamp(max=s["total"] - 1)].view(n, mq, hk, h // hk, d).permute(0, 2, 3, 1, 4)
    k = s["k"][kj].float().masked_fill(~k_ok[:, :, None, None], 0).permute(0, 2, 3, 1)
    v = s["v"][kj].float().masked_fill(~k_ok[:, :, None, None], 0).permute(0, 2, 1, 3)
    x = torch.matmul(q.reshape(n, hk, (h // hk) * mq, d), k).view(n, hk, h // hk, mq, mk) * s["scale"]
    seen = k_ok[:, None, :]
    if c["causal"]:
        seen = seen & (j <= t[:, None] + (kl - ql)[:, None, None])
    x.masked_fill_(~seen[:, None, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p = x.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(n, hk, (h // hk) * mq, mk), v).view(n, hk, h // hk, mq, d) / torch.where(total > 0, total, 1.0)
    lse = (total.log() + m)[..., 0]
    at = qi.reshape(-1)
    s["out"].index_copy_(0, at, o.permute(0, 3, 1, 2, 4).reshape(n * mq, h, d).to(s["out"].dtype))
    s["lse"].index_copy_(0, at, lse.permute(0, 3, 1, 2).reshape(n * mq, h))
    return {"out": s["out"][:s["total"]], "lse": s["lse"][:s["total"]]}


def _own_attention(s):
    from tacker_b200 import ops

    c = s["case"]
    h, hk, d = c["heads"], c["kv_heads"], c["dim"]
    ops.attention_packed(s["q"].data_ptr(), h * d, s["k"].data_ptr(), hk * d, s["v"].data_ptr(), hk * d,
                         s["out"].data_ptr(), h * d, s["lse"].data_ptr(), CODES[c["type"]], s["q_start"].data_ptr(),
                         s["k_start"].data_ptr(), s["k_len"].data_ptr(), c["seqs"], s["total"], s["rows"], s["max_q"],
                         s["max_k"], h, hk, d, s["scale"], c["causal"], s["workspace"].data_ptr(), WORKSPACE_BYTES,
                         stream=torch.cuda.current_stream().cuda_stream)
    return {"out": s["out"][:s["total"]], "lse": s["lse"][:s["total"]]}


def _rope(s):
    c = s["case"]
    t, h, hk, d, rot = c["tokens"], c["heads"], c["kv_heads"], c["dim"], c["rot"]
    x = s["x"].float()
    if s["bias"] is not None:
        x = x + s["bias"]
    x = x.view(t, h + 2 * hk, d)
    a = s["pos"].double()[:, None] * s["turns"]
    a = (a - a.round()) * (2 * math.pi)
    cos, sin = ((f(a) * c["magnitude"]).float()[:, None, :] for f in (torch.cos, torch.sin))
    qk = x[:, :h + hk]
    if c["interleaved"]:
        u, w = qk[..., 0:rot:2], qk[..., 1:rot:2]
        turned = torch.stack((u * cos - w * sin, w * cos + u * sin), -1).flatten(-2)
    else:
        u, w = qk[..., :rot // 2], qk[..., rot // 2:rot]
        turned = torch.cat((u * cos - w * sin, w * cos + u * sin), -1)
    qk = torch.cat((turned, qk[..., rot:]), -1).to(s["q"].dtype)
    s["q"].copy_(qk[:, :h])
    if s["slots"] is None:
        s["k"].copy_(qk[:, h:])
        s["v"].copy_(x[:, h + hk:])
    else:
        s["k"].index_copy_(0, s["slots"], qk[:, h:])
        s["v"].index_copy_(0, s["slots"], x[:, h + hk:].to(s["v"].dtype))
    return {"q": s["q"], "k": s["k"], "v": s["v"]}


def _own_rope(s):
    from tacker_b200 import ops

    c = s["case"]
    h, hk, d = c["heads"], c["kv_heads"], c["dim"]
    at = lambda x: 0 if x is None else x.data_ptr()  # noqa: E731
    ops.rope_qkv(s["x"].data_ptr(), CODES[c["x_type"]], (h + 2 * hk) * d, at(s["bias"]), s["pos"].data_ptr(),
                 s["turns"].data_ptr(), c["rot"], c["interleaved"], c["magnitude"], c["tokens"], h, hk, d,
                 s["q"].data_ptr(), h * d, s["k"].data_ptr(), hk * d, s["v"].data_ptr(), hk * d, CODES[c["out_type"]],
                 at(s["slots"]), c["slots"], stream=torch.cuda.current_stream().cuda_stream)
    return {"q": s["q"], "k": s["k"], "v": s["v"]}


def _normed(v, gamma, beta, kind, eps):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps) * gamma
    return v if beta is None else v + beta


def _norm(s):
    c = s["case"]
    a = s["a"].float()
    if c["post"]:
        a = _normed(a, s["post_gamma"], s["post_beta"], c["kind"], c["eps"])
    if s["gate"] is not None:
        rows = torch.arange(c["rows"], device=a.device) // (c["gate_rows"] or c["rows"])
        a = a * s["gate"][rows]
    y = s["x"].float() + c["scale"] * a
    s["y"].copy_(y)
    if c["pre"]:
        s["h"].copy_(_normed(y, s["pre_gamma"], s["pre_beta"], c["kind"], c["eps"]))
    return {"y": s["y"], "h": s["h"]}


def _own_norm(s):
    from tacker_b200 import ops

    c = s["case"]
    n = c["cols"]
    at = lambda x: 0 if x is None else x.data_ptr()  # noqa: E731
    ops.norm_residual_rows(s["a"].data_ptr(), CODES[c["a_type"]], n, c["post"], at(s["post_gamma"]), at(s["post_beta"]),
                           at(s["gate"]), n, c["gate_rows"] if c["gate_rows"] > 0 else c["rows"], c["scale"],
                           s["x"].data_ptr(), n, s["y"].data_ptr(), n, CODES[c["x_type"]], at(s["pre_gamma"]),
                           at(s["pre_beta"]), s["h"].data_ptr() if c["pre"] else 0, n, CODES[c["h_type"]],
                           c["kind"] == "layer", c["eps"], c["rows"], n, stream=torch.cuda.current_stream().cuda_stream)
    return {"y": s["y"], "h": s["h"]}


def _i8(s):
    x = s["x"].float()
    # the quotient rounded once (torch divides an fp32 tensor by a number as a product with its rounded reciprocal)
    scale = (x.abs().amax(1).double() / 127).float()
    scale = torch.where(scale < torch.finfo(torch.float32).tiny, 0.0, scale)
    # to the nearest of the scale's multiples, in 64 bits: halves of the largest value lie next to a border
    codes = (x.double() / torch.where(scale > 0, scale, 1.0).double()[:, None]).round()
    codes = torch.where(scale[:, None] > 0, codes, 0.0).float()
    y = torch.matmul(codes, s["w"].float().t()) * scale[:, None] * s["ws"]
    if s["bias"] is not None:
        y = y + s["bias"]
    s["codes"].copy_(codes)
    s["scales"].copy_(scale)
    s["out"].copy_(y)
    return {"codes": s["codes"], "scales": s["scales"], "out": s["out"]}


def _own_i8(s):
    from tacker_b200 import ops

    c = s["case"]
    m, n, k = c["rows"], c["outs"], c["cols"]
    stream = torch.cuda.current_stream().cuda_stream
    ops.quantize_rows_i8(s["x"].data_ptr(), CODES[c["x_type"]], k, s["codes"].data_ptr(), k, s["scales"].data_ptr(), m, k,
                         stream=stream)
    ops.i8gemm(s["codes"].data_ptr(), k, s["scales"].data_ptr(), s["w"].data_ptr(), k, s["ws"].data_ptr(),
               0 if s["bias"] is None else s["bias"].data_ptr(), s["out"].data_ptr(), n, CODES[c["out_type"]], m, n, k,
               stream=stream)
    return {"codes": s["codes"], "scales": s["scales"], "out": s["out"]}


# ---- what a pass cannot do without ---------------------------------------------------------------------------------
def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if case["op"] == "attention":
        ql, kl = _lengths(case)
        pairs = 0
        for q, k in zip(ql, kl):  # keys that some query sees, over the queries
            if case["causal"]:
                first = max(0, k - q + 1)
                pairs += (first + k) * (k - first + 1) // 2
            else:
                pairs += q * k
        b = size[case["type"]]
        return {"bytes": 2 * sum(ql) * case["heads"] * case["dim"] * b + sum(ql) * case["heads"] * 4
                + 2 * sum(kl) * case["kv_heads"] * case["dim"] * b, "flops": 4 * pairs * case["heads"] * case["dim"]}
    if case["op"] == "rope":
        n = (case["heads"] + 2 * case["kv_heads"]) * case["dim"]
        return {"bytes": case["tokens"] * (n * (size[case["x_type"]] + size[case["out_type"]]) + 4 + 8 * bool(case["slots"]))
                + 4 * n * case["bias"], "flops": 3 * case["tokens"] * (case["heads"] + case["kv_heads"]) * case["rot"]}
    if case["op"] == "norm":
        n = case["rows"] * case["cols"]
        gates = {-1: 0, 0: 1}.get(case["gate_rows"], -(-case["rows"] // max(1, case["gate_rows"])))
        return {"bytes": n * (size[case["a_type"]] + 2 * size[case["x_type"]] + size[case["h_type"]] * case["pre"])
                + 4 * case["cols"] * (gates + case["post"] + case["pre"]), "flops": n * 12}
    m, n, k = case["rows"], case["outs"], case["cols"]
    return {"bytes": m * k * (size[case["x_type"]] + 1) + n * k + m * n * size[case["out_type"]] + 4 * (m + n),
            "flops": 2 * m * n * k}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attention":
        ql, kl = _lengths(case)
        group = case["heads"] // case["kv_heads"]
        out = torch.zeros(s["total"], case["heads"], case["dim"], dtype=torch.float64, device="cuda")
        lse = torch.zeros(s["total"], case["heads"], dtype=torch.float64, device="cuda")
        first = 0
        for i, (n, m) in enumerate(zip(ql, kl)):
            k0 = int(s["k_start"][i])
            hidden = torch.ones(n, m, dtype=torch.bool, device="cuda").triu(m - n + 1) if case["causal"] else None
            for h in range(case["heads"]):
                q = s["q"][first:first + n, h].double()
                k, v = (s[w][k0:k0 + m, h // group].double() for w in "kv")
                z = (q @ k.t()) * s["scale"]
                if hidden is not None:
                    z[hidden] = -math.inf
                total = torch.logsumexp(z, 1)
                lse[first:first + n, h] = total
                out[first:first + n, h] = torch.exp(z - torch.where(total == -math.inf, 0.0, total)[:, None]) @ v
            first += n
        return {"out": out, "lse": lse}
    if case["op"] == "rope":
        h, hk, d, rot = case["heads"], case["kv_heads"], case["dim"], case["rot"]
        x = s["x"].double()
        if s["bias"] is not None:
            x = x + s["bias"].double()
        x = x.view(case["tokens"], h + 2 * hk, d).clone()
        angle = 2 * math.pi * torch.frac(s["pos"].double()[:, None] * s["turns"][None, :])
        turn = torch.polar(torch.full_like(angle, case["magnitude"]), angle)[:, None, :]
        even, odd = (slice(0, rot, 2), slice(1, rot, 2)) if case["interleaved"] else (slice(0, rot // 2), slice(rot // 2, rot))
        z = torch.complex(x[:, :h + hk, even], x[:, :h + hk, odd]) * turn
        x[:, :h + hk, even], x[:, :h + hk, odd] = z.real, z.imag
        k, v = (torch.zeros(*s["k"].shape, dtype=torch.float64, device="cuda") for _ in "kv")
        at = torch.arange(case["tokens"], device="cuda") if s["slots"] is None else s["slots"]
        k[at], v[at] = x[:, h:h + hk], x[:, h + hk:]
        return {"q": x[:, :h].contiguous(), "k": k, "v": v}
    if case["op"] == "norm":
        def norm(z, gamma, beta):
            mean = z.mean(1, keepdim=True) if case["kind"] == "layer" else 0.0
            z = (z - mean) * torch.rsqrt((z - mean).square().mean(1, keepdim=True) + case["eps"]) * gamma.double()
            return z if beta is None else z + beta.double()

        branch = s["a"].double()
        if case["post"]:
            branch = norm(branch, s["post_gamma"], s["post_beta"])
        if s["gate"] is not None:
            branch = branch * s["gate"].double().repeat_interleave(case["gate_rows"] or case["rows"], 0)[:case["rows"]]
        y = s["x"].double() + case["scale"] * branch
        return {"y": y, "h": norm(y, s["pre_gamma"], s["pre_beta"]) if case["pre"] else torch.zeros_like(y)}
    scale = s["x"].double().abs().max(1).values.div(127).float()  # kept in 32 bits: that is part of the definition
    scale[scale < 2.0 ** -126] = 0
    codes = torch.nan_to_num(torch.round(s["x"].double() / scale.double()[:, None]), nan=0.0)
    out = (codes @ s["w"].double().t()) * (scale.double()[:, None] * s["ws"].double()[None, :])
    if s["bias"] is not None:
        out = out + s["bias"].double()
    return {"codes": codes.to(torch.int8), "scales": scale, "out": out}
