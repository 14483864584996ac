"""The mixture-of-experts operators with 8-bit weights and activations: what is measured of them.

Four operators of one expert layer, in the order in which a layer runs them:

* the block quantiser (`block_quant_fp8`, `swiglu_block_quant_fp8`): fp8 codes with one fp32 scale per 128 values;
* the token permutation (`moe_token_permute`, `moe_token_permute_grad`): tokens sorted by expert, and its gradient;
* the block-scaled fp8 matrix product, dense and over experts (`block_quant_matmul`, `block_quant_grouped_matmul`);
* the way back (`moe_token_unpermute`, `moe_token_unpermute_grad`): weighted sums per token, and their gradients.

A case is a dict; `op` says which operator it runs.  Where `own` is false `run` computes the operator in elementary torch
operations in 32 bits, else it calls the package.
"""
import math

import numpy as np
import torch

own = False

FP8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
FP8_MAX = {"e4m3": 448.0, "e5m2": 57344.0}
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4, "e4m3": 1, "e5m2": 1}
BLK = 128
TINY = 2.0 ** -126


def listed():
    return [
        # the activations of a few decoding requests in front of an fp8 projection: launch latency
        dict(name="quant decode", op="quant", rows=8, d=4096, type="bf16", code="e4m3"),
        # the gated activations of a prefill batch, odd row count: bandwidth
        dict(name="swiglu quant prefill", op="swiglu", rows=4099, d=14336, type="bf16", code="e4m3"),
        # one token through an up-projection stored [N, K]: the weight stream
        dict(name="matmul one token", op="matmul", m=1, k=4096, n=14336, nk=True, x="e4m3", out="bf16"),
        # a ragged batch on a weight stored [K, N], no size a multiple of a tile
        dict(name="matmul ragged", op="matmul", m=77, k=4112, n=2000, nk=False, x="e5m2", out="fp16"),
        # a long prefill through a large projection: tensor rate
        dict(name="matmul prefill", op="matmul", m=4096, k=8192, n=28672, nk=True, x="e4m3", out="bf16"),
        # a decode batch over many experts: a few rows each, some experts empty
        dict(name="grouped decode", op="grouped", tokens=32, topk=8, experts=64, k=2048, n=2816, nk=True, x="e4m3", out="bf16"),
        # a prefill over few experts, uneven loads
        dict(name="grouped prefill", op="grouped", tokens=4096, topk=2, experts=8, k=4096, n=14336, nk=True, x="e4m3", out="bf16"),
        # the dispatch of a decode batch: launch latency
        dict(name="permute decode", op="permute", tokens=16, topk=8, experts=64, h=4096, type="bf16", away=0),
        # the dispatch of quantised prefill tokens with their scales, a part of the experts elsewhere
        dict(name="permute prefill", op="permute", tokens=8191, topk=8, experts=256, h=4096, type="e4m3", away=25),
        # its gradient in training
        dict(name="permute gradient", op="permute_grad", tokens=4099, topk=4, experts=16, h=4096, type="fp16", away=0),
        # the weighted return of a prefill batch
        dict(name="unpermute prefill", op="unpermute", tokens=8191, topk=8, experts=256, h=4096, type="bf16", away=25),
        # its gradients in training: rows and weights
        dict(name="unpermute gradient", op="unpermute_grad", tokens=4096, topk=8, experts=64, h=4096, type="bf16", away=0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["quant", "swiglu", "matmul", "matmul", "grouped", "grouped", "permute", "permute_grad", "unpermute", "unpermute_grad"])
    if op in ("quant", "swiglu"):
        d = _log(rng, 64, 16384)
        d -= d % rng.choice([1, 8, 128])
        return dict(op=op, rows=_log(rng, 1, max(1, min(8192, (60 << 20) // max(d, 1)))), d=max(d, 8), type=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                    code=rng.choice(["e4m3", "e4m3", "e5m2"]))
    if op == "matmul":
        k, n = 16 * _log(rng, 8, 512), 16 * _log(rng, 8, 1024)
        return dict(op=op, m=_log(rng, 1, 4096), k=k, n=n, nk=rng.random() < 0.6, x=rng.choice(["e4m3", "e4m3", "e5m2"]), out=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    if op == "grouped":
        e, topk = rng.choice([4, 8, 16, 32, 60, 64, 128]), rng.choice([1, 2, 4, 6, 8])
        k, n = 16 * _log(rng, 16, 256), 16 * _log(rng, 16, 512)
        while e * k * n > 450 << 20:
            k, n = max(256, k // 2 // 16 * 16), max(256, n // 2 // 16 * 16)
        return dict(op=op, tokens=_log(rng, 1, 4096), topk=min(topk, e), experts=e, k=k, n=n, nk=rng.random() < 0.7, x="e4m3", out=rng.choice(["bf16", "bf16", "fp16"]))
    e, topk = rng.choice([4, 8, 16, 60, 64, 128, 256]), rng.choice([1, 2, 4, 6, 8])
    h = _log(rng, 64, 8192)
    h -= h % rng.choice([1, 8, 128])
    types = ["bf16", "bf16", "fp16", "fp32"] + (["e4m3"] if op == "permute" else [])
    return dict(op=op, tokens=_log(rng, 1, max(1, min(8191, (48 << 20) // (h * min(topk, e))))), topk=min(topk, e), experts=e, h=max(h, 16),
                type=rng.choice(types), away=rng.choice([0, 0, 25]))


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _activations(g, rows, d, dt):
    # activations have a few channels far above the others
    x = torch.randn((rows, d), generator=g, device="cuda")
    x *= torch.exp(0.8 * torch.randn((d,), generator=g, device="cuda"))
    return x.to(dt)


def _codes_of_rows(x, code):
    """fp8 codes and scales [rows, ceil(d / 128)] of activations, as the quantiser in front of a product makes them."""
    rows, d = x.shape
    kb = -(-d // BLK)
    v = torch.zeros((rows, kb * BLK), device="cuda")
    v[:, :d] = x
    v = v.view(rows, kb, BLK)
    s = (v.abs().amax(-1) / FP8_MAX[code]).clamp_min(1e-20)
    q = (v * (1.0 / s).unsqueeze(-1)).to(FP8[code]).view(rows, kb * BLK)
    return q.view(torch.uint8)[:, :d].contiguous().view(FP8[code]), s


def _weights(g, e, k, n, nk):
    """e4m3 weights [e, n, k] (nk) or [e, k, n], and their scales per 128 x 128 block in the same order."""
    a, b = (n, k) if nk else (k, n)
    ab, bb = -(-a // BLK), -(-b // BLK)
    q = torch.empty((e, a, b), dtype=torch.uint8, device="cuda")
    s = torch.empty((e, ab, bb), device="cuda")
    for i in range(e):
        w = torch.zeros((ab * BLK, bb * BLK), device="cuda")
        w[:a, :b] = torch.randn((a, b), generator=g, device="cuda") * (0.02 * math.exp(0.2 * (i % 5)))
        w = w.view(ab, BLK, bb, BLK)
        s[i] = (w.abs().amax((1, 3)) / 448.0).clamp_min(1e-20)
        c = (w * (1.0 / s[i])[:, None, :, None]).to(torch.float8_e4m3fn).view(torch.uint8).view(ab * BLK, bb * BLK)
        q[i] = c[:a, :b]
    return q.view(torch.float8_e4m3fn), s


def _routing(case, seed):
    """Experts of each token, the nearest first, with uneven loads; `away` per cent of the experts are on other machines (id -1)."""
    r = np.random.RandomState(int(seed) % (1 << 31))
    t, e, k = case["tokens"], case["experts"], case["topk"]
    score = r.standard_normal((t, e)) + 0.7 * r.standard_normal(e)
    ids = np.argsort(-score, axis=1, kind="stable")[:, :k].copy()
    top = np.take_along_axis(score, ids, 1)
    probs = np.exp(top - top.max(1, keepdims=True))
    probs /= probs.sum(1, keepdims=True)
    ids[ids >= e - e * case.get("away", 0) // 100] = -1
    return ids, probs.astype(np.float32)


def _order(ids, e):
    """Where each (token, choice) lands when they are sorted by expert, earlier tokens first; -1 for those that are away; rows per expert."""
    flat = ids.reshape(-1)
    key = np.where(flat < 0, e, flat)
    order = np.argsort(key, kind="stable")
    place = np.empty(flat.size, dtype=np.int32)
    place[order] = np.arange(flat.size, dtype=np.int32)
    place[flat < 0] = -1
    return place.reshape(ids.shape), np.bincount(key, minlength=e + 1)[:e].astype(np.int64)


def prepare(case, seed):
    g, op, c = _gen(seed), case["op"], case
    if op == "quant":
        return dict(case=c, x=_activations(g, c["rows"], c["d"], DT[c["type"]]))
    if op == "swiglu":
        return dict(case=c, x=_activations(g, c["rows"], 2 * c["d"], DT[c["type"]]))
    if op == "matmul":
        x, xs = _codes_of_rows(_activations(g, c["m"], c["k"], torch.float32), c["x"])
        w, ws = _weights(g, 1, c["k"], c["n"], c["nk"])
        return dict(case=c, x=x, xs=xs, w=w[0], ws=ws[0])
    ids, probs = _routing(c, seed)
    place, counts = _order(ids, c["experts"])
    rows = c["tokens"] * c["topk"]
    if op == "grouped":
        x, xs = _codes_of_rows(_activations(g, rows, c["k"], torch.float32), c["x"])
        w, ws = _weights(g, c["experts"], c["k"], c["n"], c["nk"])
        return dict(case=c, x=x, xs=xs, w=w, ws=ws, counts=torch.from_numpy(counts).cuda(), most=int(counts.max()))
    st = dict(case=c, place=torch.from_numpy(place).cuda(), probs=torch.from_numpy(probs).cuda())
    dt = torch.float32 if c["type"] == "e4m3" else DT[c["type"]]
    if op == "permute":
        st["ids"] = torch.from_numpy(ids.astype(np.int32)).cuda()
        x = _activations(g, c["tokens"], c["h"], dt)
        if c["type"] == "e4m3":
            st["x"], st["xs"] = _codes_of_rows(x, "e4m3")
            st["out_s"] = torch.zeros((rows, st["xs"].shape[1]), device="cuda")
        else:
            st["x"] = x
        # the receive buffer of the layer, whose last rows stay empty when experts are away
        st["out"] = torch.zeros((rows, c["h"]), dtype=torch.uint8 if c["type"] == "e4m3" else dt, device="cuda").view(st["x"].dtype)
    else:
        st["rows"] = torch.randn((rows, c["h"]), generator=g, device="cuda").to(dt)
        if op == "unpermute_grad":
            st["dout"] = torch.randn((c["tokens"], c["h"]), generator=g, device="cuda").to(dt)
            st["out"] = torch.zeros((rows, c["h"]), dtype=dt, device="cuda")
    return st


# ------------------------------------------------------------------------------------------------ one pass
_package = None


def _pkg():
    global _package
    if _package is None:
        import __graft_entry__
        _package = __graft_entry__.load_package()
    return _package


def run(st):
    return _run_own(st) if own else _run_plain(st)


def _run_own(st):
    p, c, op = _pkg(), st["case"], st["case"]["op"]
    if op == "quant":
        return p.block_quant_fp8(st["x"], dtype=FP8[c["code"]])
    if op == "swiglu":
        return p.swiglu_block_quant_fp8(st["x"], dtype=FP8[c["code"]])
    if op == "matmul":
        return p.block_quant_matmul(st["x"], st["xs"], st["w"], st["ws"], transposed=c["nk"], out_dtype=DT[c["out"]])
    if op == "grouped":
        return p.block_quant_grouped_matmul(st["x"], st["xs"], st["w"], st["ws"], st["counts"], transposed=c["nk"], out_dtype=DT[c["out"]])
    if op == "permute":
        return p.moe_token_permute(st["x"], st["ids"], c["experts"], scales=st.get("xs"), out=st["out"], scales_out=st.get("out_s"))
    if op == "permute_grad":
        return p.moe_token_permute_grad(st["rows"], st["place"])
    if op == "unpermute":
        return p.moe_token_unpermute(st["rows"], st["place"], st["probs"])
    return p.moe_token_unpermute_grad(st["dout"], st["rows"], st["place"], st["probs"], out=st["out"])


def _plain_quant(v, code):
    rows, d = v.shape
    kb = -(-d // BLK)
    if d % BLK:
        v = torch.cat([v, v.new_zeros((rows, kb * BLK - d))], 1)
    v = v.view(rows, kb, BLK)
    top = v.abs().amax(-1)
    s = torch.where(top > 0, (top / FP8_MAX[code]).clamp_min(TINY), torch.ones_like(top))
    q = (v * (1.0 / s).unsqueeze(-1)).to(FP8[code]).view(torch.uint8).view(rows, kb * BLK)
    return q[:, :d].contiguous().view(FP8[code]), s


def _wide(s, size):
    return s.repeat_interleave(BLK, -1)[..., :size]


def _plain_weight(w, ws):
    a, b = w.shape[-2], w.shape[-1]
    return w.float() * _wide(ws, b).repeat_interleave(BLK, -2)[..., :a, :]


def _run_plain(st):
    c, op = st["case"], st["case"]["op"]
    if op == "quant":
        return _plain_quant(st["x"].float(), c["code"])
    if op == "swiglu":
        a, b = st["x"].float().chunk(2, -1)
        return _plain_quant(a / (1.0 + torch.exp(-a)) * b, c["code"])
    if op == "matmul":
        x = st["x"].float() * _wide(st["xs"], c["k"])
        w = _plain_weight(st["w"], st["ws"])
        return (x @ (w.t() if c["nk"] else w)).to(DT[c["out"]])
    if op == "grouped":
        # the rows of each expert in a batch of their own, padded to the largest
        x = st["x"].float() * _wide(st["xs"], c["k"])
        w = _plain_weight(st["w"], st["ws"])
        ends = st["counts"].cumsum(0)
        r = torch.arange(x.shape[0], device=x.device)
        e = torch.searchsorted(ends, r, right=True)
        at = r - (ends - st["counts"])[e]
        pad = x.new_zeros((c["experts"], st["most"], c["k"]))
        pad[e, at] = x
        return torch.bmm(pad, w.transpose(1, 2) if c["nk"] else w)[e, at].to(DT[c["out"]])
    if op == "permute":
        # a stable sort of (token, choice) by expert; what is away sorts last and is not written
        flat = st["ids"].reshape(-1).long()
        key = torch.where(flat < 0, torch.full_like(flat, c["experts"]), flat)
        order = torch.sort(key, stable=True).indices
        place = torch.empty_like(order)
        place[order] = torch.arange(order.numel(), device=order.device)
        place = torch.where(flat < 0, torch.full_like(place, -1), place)
        counts = torch.zeros(c["experts"] + 1, dtype=torch.int64, device=flat.device).index_add_(0, key, torch.ones_like(key))[:c["experts"]]
        keep = (torch.arange(order.numel(), device=order.device) < counts.sum()).unsqueeze(1)
        src = order // c["topk"]
        fp8 = c["type"] == "e4m3"
        x, out = (st["x"].view(torch.uint8), st["out"].view(torch.uint8)) if fp8 else (st["x"], st["out"])
        out = torch.where(keep, x[src], out)
        place = place.view(st["ids"].shape).to(torch.int32)
        if fp8:
            return out.view(st["x"].dtype), place, counts, torch.where(keep, st["xs"][src], st["out_s"])
        return out, place, counts
    rows, place = st["rows"].float(), st["place"].long()
    there = (place >= 0).unsqueeze(-1)
    if op in ("permute_grad", "unpermute"):
        v = torch.where(there, rows[place.clamp_min(0)], rows.new_zeros(()))
        if op == "unpermute":
            v = v * st["probs"].unsqueeze(-1)
        return v.sum(1).to(st["rows"].dtype)
    dout = st["dout"].float().unsqueeze(1)
    v = torch.where(there, rows[place.clamp_min(0)], rows.new_zeros(()))
    dprobs = (dout * v).sum(-1)
    drows = (st["probs"].unsqueeze(-1) * dout).reshape(-1, rows.shape[1])
    there = there.reshape(-1)
    out = st["out"].clone()
    out[place.reshape(-1)[there]] = drows[there].to(st["rows"].dtype)
    return out, dprobs


# ------------------------------------------------------------------------------------------------ what it costs
def work(case):
    c, op = case, case["op"]
    if op in ("quant", "swiglu"):
        n = c["rows"] * c["d"]
        return {"bytes": n * BYTES[c["type"]] * (2 if op == "swiglu" else 1) + n + 4 * c["rows"] * -(-c["d"] // BLK), "flops": n * (10 if op == "swiglu" else 3)}
    if op in ("matmul", "grouped"):
        k, n, kb, nb = c["k"], c["n"], -(-c["k"] // BLK), -(-c["n"] // BLK)
        m = c["m"] if op == "matmul" else c["tokens"] * c["topk"]
        e = 1 if op == "matmul" else min(c["experts"], m)
        return {"bytes": m * (k + 4 * kb) + e * (k * n + 4 * kb * nb) + m * n * BYTES[c["out"]], "flops": 2 * m * n * k}
    t, k, h, b = c["tokens"], c["topk"], c["h"], BYTES[c["type"]]
    live = t * k * (100 - c["away"]) // 100
    row = h * b + (4 * -(-h // BLK) if c["type"] == "e4m3" else 0)
    if op == "permute":
        return {"bytes": t * row + live * row + 8 * t * k + 8 * c["experts"], "flops": t * k}
    if op == "unpermute_grad":
        return {"bytes": t * h * b + 2 * live * h * b + 12 * t * k, "flops": 3 * live * h}
    return {"bytes": live * h * b + t * h * b + 4 * t * k * (2 if op == "unpermute" else 1), "flops": live * h * (2 if op == "unpermute" else 1)}


# ------------------------------------------------------------------------------------------------ in 64 bits
def _exact_codes(v, top):
    """Real-valued codes v / scale and the scales; the 8-bit rounding is the output type's own."""
    rows, d = v.shape
    kb = -(-d // BLK)
    full = torch.nn.functional.pad(v, (0, kb * BLK - d)).reshape(rows, kb, BLK)
    m = full.abs().max(-1).values
    s = torch.where(m == 0, 1.0, m / top)
    return (full / s[..., None]).reshape(rows, -1)[:, :d], s


def _exact_weight(q, s):
    a, b = q.shape
    ia, ib = torch.arange(a, device=q.device) // BLK, torch.arange(b, device=q.device) // BLK
    return q.double() * s.double()[ia][:, ib]


def exact(case, seed):
    st, c, op = prepare(case, seed), case, case["op"]
    if op == "quant":
        return _exact_codes(st["x"].double(), FP8_MAX[c["code"]])
    if op == "swiglu":
        x = st["x"].double()
        return _exact_codes(x[:, :c["d"]] * torch.sigmoid(x[:, :c["d"]]) * x[:, c["d"]:], FP8_MAX[c["code"]])
    if op in ("matmul", "grouped"):
        x = st["x"].double() * st["xs"].double()[:, torch.arange(c["k"], device="cuda") // BLK]
        if op == "matmul":
            w = _exact_weight(st["w"], st["ws"])
            return torch.matmul(x, w.t() if c["nk"] else w)
        out, at = torch.zeros((x.shape[0], c["n"]), dtype=torch.float64, device="cuda"), 0
        for e, r in enumerate(st["counts"].tolist()):
            if r:
                w = _exact_weight(st["w"][e], st["ws"][e])
                out[at:at + r] = torch.matmul(x[at:at + r], w.t() if c["nk"] else w)
            at += r
        return out
    if op == "permute":
        return None
    place, rows = st["place"].cpu().numpy(), st["rows"].double()
    t, k = place.shape
    zero = torch.cat([rows, rows.new_zeros((1, rows.shape[1]))])
    picked = torch.from_numpy(np.where(place < 0, rows.shape[0], place).astype(np.int64)).cuda()
    if op in ("permute_grad", "unpermute"):
        total = rows.new_zeros((t, rows.shape[1]))
        for j in range(k):
            total += zero[picked[:, j]] * (st["probs"][:, j:j + 1].double() if op == "unpermute" else 1.0)
        return total
    dout, dp = st["dout"].double(), torch.zeros((t, k), dtype=torch.float64, device="cuda")
    out = torch.zeros_like(zero)
    for j in range(k):
        dp[:, j] = (dout * zero[picked[:, j]]).sum(1)
        out[picked[:, j]] = dout * st["probs"][:, j:j + 1].double()
    return out[:-1], dp
