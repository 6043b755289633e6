"""The block-scaled FP8 operators: what they compute in plain torch, and the calls that a program makes of them.

An FP8 linear layer keeps E4M3 elements with one fp32 scale per 128 elements of a row (activations, gradients,
checkpoints) or per 128 x 128 tile (weights).  The same quantised activations are the forward product's operand and the
checkpoint that the backward pass reads.

    quantize     activations or a weight to the format (scales are powers of two); ``restore`` = back to 16 bits as well
    gemm         C = A . B^T over such operands; ``transposed``: B stored [K, N], the form the input gradient takes
    wgrad        the weight gradient dY^T . X from 16-bit dY and 8-bit X, over one or two micro-batches
    swiglu       silu(gate) * up to the format, with the gate and up checkpoints; the result is restored to be looked at
    swiglu_bwd   the gradients of gate and up from the checkpoints
    swiglu_step  both, one after the other

Sizes are those of the benchmark configurations (65536 tokens, d_model 512, feed-forward 2048, QKV 1536) and of the tests.
"""
import math

import torch

own = False
DEV = "cuda"
BLOCK = 128
_DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # a full training batch through the widest forward products of a layer: QKV projection, feed-forward up (the largest N)
        dict(name="gemm_qkv_batch", op="gemm", M=65536, N=1536, K=512, dtype="f16", transposed=False),
        # the down-projection of a batch of 9001 tokens, bf16, N that is no multiple of a tile
        dict(name="gemm_down_ragged", op="gemm", M=9001, N=520, K=2048, dtype="bf16", transposed=False),
        # one token of a decoder through the feed-forward's first product: latency
        dict(name="gemm_token", op="gemm", M=1, N=2048, K=512, dtype="f16", transposed=False),
        # input gradient of the feed-forward's first product: the weight as the forward pass has it, reduced over its rows
        dict(name="gemm_dgrad_batch", op="gemm", M=65536, N=512, K=2048, dtype="bf16", transposed=True),
        # weight gradient of the feed-forward's first product over a full batch, from the 8-bit checkpoint of its input
        dict(name="wgrad_batch", op="wgrad", M=65536, N=2048, K=512, dtype="bf16", micro=1),
        # a ragged batch accumulated over two micro-batches, fp16
        dict(name="wgrad_micro_ragged", op="wgrad", M=9001, N=1000, K=520, dtype="f16", micro=2),
        # the activations of a full batch (a layer's input), and a master weight after an optimizer step
        dict(name="quantize_batch", op="quantize", M=65536, K=512, dtype="bf16", rows=1, restore=False),
        dict(name="quantize_weight", op="quantize", M=2048, K=512, dtype="f32", rows=128, restore=False),
        # a checkpoint packed and restored, odd row length
        dict(name="checkpoint_ragged", op="quantize", M=20001, K=1001, dtype="f16", rows=1, restore=True),
        # the feed-forward's activation, forward and backward, over a full batch
        dict(name="swiglu_batch", op="swiglu", M=65536, F=2048, dtype="bf16"),
        dict(name="swiglu_bwd_batch", op="swiglu_bwd", M=65536, F=2048, dtype="bf16"),
        # both for a few hundred tokens of an odd width: launches count
        dict(name="swiglu_step_small", op="swiglu_step", M=333, F=1000, dtype="f16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A layer's width: whole blocks, a multiple of 8, or odd."""
    n = _log(rng, lo, hi)
    how = rng.random()
    return max(BLOCK, n // BLOCK * BLOCK) if how < 0.4 else max(8, n // 8 * 8) if how < 0.7 else n


def draw(rng):
    op = rng.choice(["gemm", "gemm", "gemm", "wgrad", "wgrad", "quantize", "swiglu", "swiglu_bwd", "swiglu_step"])
    most = 65536 * 1536 * 512
    if op == "gemm" or op == "wgrad":
        n, k = _width(rng, 64, 4096), _width(rng, 64, 4096)
        m = _log(rng, 1, min(65536, most // (n * k)))
        if op == "gemm":
            return dict(op=op, M=m, N=n, K=k, dtype=rng.choice(["f16", "bf16", "f32"]), transposed=rng.random() < 0.4)
        return dict(op=op, M=m, N=n, K=k, dtype=rng.choice(["f16", "bf16"]), micro=rng.choice([1, 1, 2]))
    w = _width(rng, 64, 4096)
    m = _log(rng, 1, min(65536, 65536 * 1024 // w))
    if op == "quantize":
        rows = rng.choice([1, 1, 128])
        return dict(op=op, M=m, K=w, dtype=rng.choice(["f16", "bf16", "f32"]), rows=rows, restore=rng.random() < 0.5)
    return dict(op=op, M=m, F=w, dtype=rng.choice(["f16", "bf16", "f32"]))


# ---- the format in plain torch ---------------------------------------------------------------------------------------
def _blocks(x, rows):
    """[M, K] fp32 -> [M / rows, rows, K / 128, 128], zero-padded to whole blocks."""
    m, k = x.shape
    x = torch.nn.functional.pad(x, (0, -k % BLOCK, 0, -m % rows))
    return x.view(x.shape[0] // rows, rows, x.shape[1] // BLOCK, BLOCK)


def _quantize(x, rows):
    m, k = x.shape
    b = _blocks(x.float(), rows)
    amax = torch.where(torch.isfinite(b), b.abs(), 0.0).amax(dim=(1, 3))
    mant, expo = torch.frexp(amax)                      # amax = mant 2^expo, 448 = 0.875 2^9
    expo = torch.where(mant <= 0.875, expo - 9, expo - 8).clamp(min=-126)
    s = torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), expo), 1.0)
    q = (b / s[:, None, :, None]).reshape(b.shape[0] * rows, -1)[:m, :k].to(torch.float8_e4m3fn)
    return q, s


def _spread(s, rows, m, k):
    """The scale of every element."""
    return s.repeat_interleave(rows, 0)[:m].repeat_interleave(BLOCK, 1)[:, :k]


def _restore(q, s, rows):
    return q.float() * _spread(s, rows, *q.shape)


# ---- inputs ------------------------------------------------------------------------------------------------------------
def _rows16(q):
    """Rows on 16-byte boundaries, as the quantisers lay them out."""
    m, k = q.shape
    buf = torch.zeros((m, (k + 15) // 16 * 16), dtype=torch.uint8, device=q.device)
    buf[:, :k] = q.view(torch.uint8)
    return buf.view(torch.float8_e4m3fn)[:, :k]


def _pad8(x):
    m, k = x.shape
    buf = torch.zeros((m, (k + 7) // 8 * 8), dtype=x.dtype, device=x.device)
    buf[:, :k] = x
    return buf[:, :k]


class _Rand:
    def __init__(self, seed):
        self.gen = torch.Generator(device=DEV).manual_seed(seed)

    def normal(self, m, n, std=1.0):
        return torch.randn(m, n, generator=self.gen, device=DEV) * std

    def act(self, m, n):                        # activations: N(0, 1) with a few channels that are ten times as large
        loud = 1 + 9 * (torch.rand(n, generator=self.gen, device=DEV) < 0.02).float()
        return self.normal(m, n) * loud


def prepare(case, seed):
    r, op, dt = _Rand(seed), case["op"], _DT[case["dtype"]]
    st = dict(case)
    m = case["M"]
    if op == "gemm":
        n, k = case["N"], case["K"]
        a, sa = _quantize(r.act(m, k), 1)
        w = r.normal(n, k, k ** -0.5)
        b, sb = _quantize(w.t().contiguous() if case["transposed"] else w, BLOCK)
        # scales of a published weight are any fp32 numbers, not powers of two
        sb = sb * (0.75 + 0.5 * torch.rand(sb.shape, generator=r.gen, device=DEV))
        st.update(a=_rows16(a), sa=sa, b=_rows16(b), sb=sb)
    elif op == "wgrad":
        x, sx = _quantize(r.act(m * case["micro"], case["K"]), 1)
        dy = r.normal(m * case["micro"], case["N"], 1e-2).to(dt)
        st.update(x=_rows16(x).split(m), sx=sx.split(m), dy=_pad8(dy).split(m))
    elif op == "quantize":
        x = r.normal(m, case["K"], 0.05) if case["rows"] == BLOCK else r.act(m, case["K"])
        st.update(x=_pad8(x.to(dt)))
    else:
        f = case["F"]
        st.update(gate=_pad8(r.act(m, f).to(dt)), up=_pad8(r.normal(m, f).to(dt)), dh=_pad8(r.normal(m, f, 1e-2).to(dt)))
        if op == "swiglu_bwd":
            (gq, gs), (uq, us) = _quantize(st.pop("gate"), 1), _quantize(st.pop("up"), 1)
            st.update(gq=_rows16(gq), gs=gs, uq=_rows16(uq), us=us)
    return st


# ---- one pass -----------------------------------------------------------------------------------------------------------
def _bwd(dh, gq, gs, uq, us):
    g, u, d = _restore(gq, gs, 1), _restore(uq, us, 1), dh.float()
    sig = 1 / (1 + torch.exp(-g))
    return (d * u * sig * (1 + g * (1 - sig))).to(dh.dtype), (d * g * sig).to(dh.dtype)


def _fwd(gate, up):
    g = gate.float()
    return _quantize(g / (1 + torch.exp(-g)) * up.float(), 1), _quantize(gate, 1), _quantize(up, 1)


def run(st):
    return (_own if own else _plain)(st, st["op"], _DT[st["dtype"]])


def _plain(st, op, dt):
    if op == "gemm":
        b = _restore(st["b"], st["sb"], BLOCK)
        return (_restore(st["a"], st["sa"], 1) @ (b if st["transposed"] else b.t())).to(dt)
    if op == "wgrad":
        return sum(dy.float().t() @ _restore(x, s, 1) for dy, x, s in zip(st["dy"], st["x"], st["sx"]))
    if op == "quantize":
        q, s = _quantize(st["x"], st["rows"])
        return (q, s, _restore(q, s, st["rows"]).to(torch.bfloat16)) if st["restore"] else (q, s)
    if op == "swiglu_bwd":
        return _bwd(st["dh"], st["gq"], st["gs"], st["uq"], st["us"])
    h, g, u = _fwd(st["gate"], st["up"])
    h = _restore(*h, 1).to(torch.bfloat16)
    return (h, *g, *u) if op == "swiglu" else (h, *_bwd(st["dh"], *g, *u))


def _own(st, op, dt):
    import gigaslop_b200 as g
    if op == "gemm":
        return g.gemm_fp8_block(st["a"], st["b"], st["sa"], st["sb"], dtype=dt, b_transposed=st["transposed"])
    if op == "wgrad":
        out = g.gemm_fp8_block_wgrad(st["dy"][0], st["x"][0], st["sx"][0])
        for dy, x, s in zip(st["dy"][1:], st["x"][1:], st["sx"][1:]):
            g.gemm_fp8_block_wgrad(dy, x, s, out=out, accumulate=True)
        return out
    if op == "quantize":
        q, s = g.fp8_block_quantize(st["x"], rows=st["rows"])
        return (q, s, g.fp8_block_dequantize(q, s, rows=st["rows"], dtype=torch.bfloat16)) if st["restore"] else (q, s)
    if op == "swiglu_bwd":
        return g.swiglu_fp8_block_bwd(st["dh"], st["gq"], st["gs"], st["uq"], st["us"])
    (h, hs), gate, up = g.swiglu_fp8_block(st["gate"], st["up"])
    h = g.fp8_block_dequantize(h, hs, dtype=torch.bfloat16)
    return (h, *gate, *up) if op == "swiglu" else (h, *g.swiglu_fp8_block_bwd(st["dh"], *gate, *up))


# ---- from the definition, in 64 bits ------------------------------------------------------------------------------------
def _values(q, s, rows):
    """q times the scale of its block, element by element."""
    m, k = q.shape
    i = torch.arange(m, device=DEV) // rows
    j = torch.arange(k, device=DEV) // BLOCK
    return q.double() * s.double()[i[:, None], j[None, :]]


def _nearest(x, rows):
    """(scaled elements, scales) of the format, both in 64 bits: scale 2^t with the least t that keeps |x| / 2^t <= 448, elements rounded
    half to even to 4 significant bits, and to multiples of 2^-9."""
    m, k = x.shape
    x = x.double()
    mb, kb = (m + rows - 1) // rows, (k + BLOCK - 1) // BLOCK
    i = (torch.arange(m, device=DEV) // rows)[:, None]
    j = (torch.arange(k, device=DEV) // BLOCK)[None, :]
    top = torch.zeros(mb * kb, dtype=torch.float64, device=DEV)
    top.scatter_reduce_(0, (i * kb + j).reshape(-1), x.abs().reshape(-1), "amax")
    t = torch.floor(torch.log2(top.clamp(min=2.0 ** -140))) - 10
    t = t + (torch.exp2(t) * 448 < top) + (torch.exp2(t + 1) * 448 < top) + (torch.exp2(t + 2) * 448 < top)
    s = torch.where(top > 0, torch.exp2(t.clamp(min=-126)), 1.0).view(mb, kb)
    v = x / s[i, j]
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(v / step) * step, s


def exact(case, seed):
    st = prepare(case, seed)
    op = st["op"]
    if op == "gemm":
        b = _values(st["b"], st["sb"], BLOCK)
        return torch.einsum("mk,kn->mn" if st["transposed"] else "mk,nk->mn", _values(st["a"], st["sa"], 1), b)
    if op == "wgrad":
        dy, x, s = (torch.cat(st[n]) for n in ("dy", "x", "sx"))
        return torch.einsum("mn,mk->nk", dy.double(), _values(x, s, 1))
    if op == "quantize":
        q, s = _nearest(st["x"], st["rows"])
        return (q, s, q * _spread(s, st["rows"], *q.shape)) if st["restore"] else (q, s)
    if op == "swiglu_bwd":
        g, u = _values(st["gq"], st["gs"], 1), _values(st["uq"], st["us"], 1)
    else:
        gate, up = st["gate"].double(), st["up"].double()
        (h, hs), (gq, gs), (uq, us) = (_nearest(v, 1) for v in (gate * torch.sigmoid(gate) * up, gate, up))
        h = h * _spread(hs, 1, *h.shape)
        if op == "swiglu":
            return h, gq, gs, uq, us
        g, u = gq * _spread(gs, 1, *gq.shape), uq * _spread(us, 1, *uq.shape)
    d, sig = st["dh"].double(), torch.sigmoid(g)
    grads = d * (u * sig * (1 + g * torch.sigmoid(-g))), d * (g * sig)
    return grads if op == "swiglu_bwd" else (h, *grads)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------
def work(case):
    op, m = case["op"], case["M"]
    size = {"f16": 2, "bf16": 2, "f32": 4}[case["dtype"]]
    nb = lambda v: (v + BLOCK - 1) // BLOCK
    fp8 = lambda rows, cols, r=1: rows * cols + 4 * nb(cols) * (rows if r == 1 else nb(rows))
    if op == "gemm":
        n, k = case["N"], case["K"]
        return {"bytes": fp8(m, k) + fp8(n, k, BLOCK) + size * m * n, "flops": 2 * m * n * k}
    if op == "wgrad":
        n, k, m = case["N"], case["K"], m * case["micro"]
        return {"bytes": size * m * n + fp8(m, k) + 4 * n * k, "flops": 2 * m * n * k}
    if op == "quantize":
        k = case["K"]
        return {"bytes": size * m * k + fp8(m, k, case["rows"]) + (2 * m * k if case["restore"] else 0), "flops": 4 * m * k}
    f = case["F"]
    fwd, bwd = 2 * size * m * f + 3 * fp8(m, f), 3 * size * m * f
    if op == "swiglu":                      # the result comes back as 16-bit values beside the two checkpoints
        return {"bytes": 2 * size * m * f + 2 * fp8(m, f) + 2 * m * f, "flops": 16 * m * f}
    if op == "swiglu_bwd":
        return {"bytes": bwd + 2 * fp8(m, f), "flops": 20 * m * f}
    return {"bytes": bwd + 2 * size * m * f + 2 * m * f, "flops": 36 * m * f}
