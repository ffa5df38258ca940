"""Cases, inputs, plain forms and 64-bit values of three operators:

  fp8     a projection with 8-bit operands: the activation is quantised to E4M3 with one power-of-two scale for each
          128 elements of a row, the weight is kept as E4M3 codes with one such scale for each 128 x 128 block
  decay   causal linear attention with a decay for each head over whole prompts (state carried in and out)
  step    the same recurrence for one token of each sequence, the state updated in place in its slot
"""
import math

import torch

own = False

DEV = "cuda"
BLOCK = 128


def listed():
    return [
        # the query/key/value projection of one token while decoding (width 2240)
        dict(name="fp8 one token qkv", op="fp8", M=1, K=2240, N=6720, bias=False, act="none", gate=False),
        # an output projection for a small odd batch of sequences (width 1152)
        dict(name="fp8 37 rows proj", op="fp8", M=37, K=1152, N=1152, bias=True, act="none", gate=False),
        # caption features through the first layer of their embedder (2304 channels in, tanh GELU)
        dict(name="fp8 600 captions", op="fp8", M=600, K=2304, N=2240, bias=True, act="gelu", gate=False),
        # the expanding projection of the feed-forward layer, one image of 4 096 tokens, SiLU
        dict(name="fp8 expand 4096", op="fp8", M=4096, K=2240, N=11200, bias=True, act="silu", gate=False),
        # the projection back, 16 384 tokens, with the block's gate and residual
        dict(name="fp8 point 16384", op="fp8", M=16384, K=5600, N=2240, bias=False, act="none", gate=True),
        # a caption-length prompt, 20 heads of 112 channels, normalised ReLU form
        dict(name="decay prompt 77", op="decay", B=1, N=77, H=20, Hk=20, D=112, dtype="bf16", relu=True, eps=1e-8, prior=False, ragged=False),
        # a padded batch of prompts on top of earlier state, two heads to a key/value head
        dict(name="decay 4x4096 ragged", op="decay", B=4, N=4096, H=16, Hk=8, D=64, dtype="bf16", relu=False, eps=0.0, prior=True, ragged=True),
        # a long video as one sequence of tokens
        dict(name="decay video 16384", op="decay", B=1, N=16384, H=20, Hk=20, D=112, dtype="bf16", relu=True, eps=1e-8, prior=False, ragged=False),
        # full-precision check of a small model, odd length
        dict(name="decay fp32 1001", op="decay", B=2, N=1001, H=8, Hk=8, D=32, dtype="fp32", relu=True, eps=1e-8, prior=True, ragged=False),
        # the 1.6B model's heads (70 of 32 channels), eight images
        dict(name="decay 8x4096 70 heads", op="decay", B=8, N=4096, H=70, Hk=70, D=32, dtype="bf16", relu=True, eps=1e-8, prior=False, ragged=False),
        # decoding one sequence
        dict(name="step 1", op="step", B=1, H=20, Hk=20, D=112, dtype="bf16", relu=True, eps=1e-8, spare=0),
        # decoding a full batch, a few rows of it padding
        dict(name="step 256", op="step", B=256, H=16, Hk=8, D=128, dtype="bf16", relu=False, eps=0.0, spare=5),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["fp8", "decay", "step"])
    if op == "fp8":
        while True:
            M, K, N = _log(rng, 1, 16384), 16 * _log(rng, 4, 400), 8 * _log(rng, 8, 1400)
            if M * K * N <= 16384 * 5600 * 2240:
                break
        return dict(op="fp8", M=M, K=K, N=N, bias=rng.random() < 0.5, act=rng.choice(["none", "silu", "gelu"]), gate=rng.random() < 0.3)
    D = 16 * rng.randint(1, 8)
    Hk = _log(rng, 1, 40)
    H = Hk * rng.choice([1, 1, 1, 2, 4])
    dtype = "fp32" if rng.random() < 0.25 else "bf16"
    relu = rng.random() < 0.6
    eps = rng.choice([0.0, 1e-8, 1e-6]) if relu else 0.0
    if op == "step":
        B = _log(rng, 1, 256)
        while B * H * D * D > 256 * 16 * 128 * 128:
            B = max(1, B // 2)
        return dict(op="step", B=B, H=H, Hk=Hk, D=D, dtype=dtype, relu=relu, eps=eps, spare=rng.randint(0, 9))
    B, N = _log(rng, 1, 8), _log(rng, 1, 16384)
    most = 8 * 4096 * 70 * 32 // (8 if dtype == "fp32" else 2)
    while B * N * H * D > most:
        N = max(1, N // 2)
    return dict(op="decay", B=B, N=N, H=H, Hk=Hk, D=D, dtype=dtype, relu=relu, eps=eps, prior=rng.random() < 0.5, ragged=rng.random() < 0.4)


def _dt(case):
    return torch.float32 if case["dtype"] == "fp32" else torch.bfloat16


def _blocks(x2d, rows):
    """|x| maxima over blocks of `rows` x 128 (padding counts as nothing): [ceil(R / rows), ceil(K / 128)]."""
    R, K = x2d.shape
    a = torch.nn.functional.pad(x2d.abs(), (0, -K % BLOCK, 0, -R % rows))
    return a.reshape(a.shape[0] // rows, rows, a.shape[1] // BLOCK, BLOCK).amax(dim=(1, 3))


def _exponent(amax):
    """The least e with amax <= 448 * 2^e, at least -126 (448 = 0.875 * 2^9)."""
    m, e = torch.frexp(amax)
    return torch.where(amax > 0, (e - 9 + (m > 0.875).to(e.dtype)), torch.full_like(e, -126)).clamp(-126, 127)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))

    def rand(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    if case["op"] == "fp8":
        M, K, N = case["M"], case["K"], case["N"]
        # activations after a normalisation, with a few channels far larger than the rest
        x = (rand(M, K) * (1 + 15 * (torch.rand(K, generator=g, device=DEV) > 0.99))).bfloat16()
        w = rand(N, K) / math.sqrt(K)
        e = _exponent(_blocks(w, BLOCK))
        wide = e.repeat_interleave(BLOCK, 0)[:N].repeat_interleave(BLOCK, 1)[:, :K]
        codes = torch.ldexp(w, -wide).to(torch.float8_e4m3fn)
        kb = e.shape[1]
        scales = torch.zeros(e.shape[0], (kb + 3) // 4 * 4, dtype=torch.uint8, device=DEV)[:, :kb]
        scales.copy_(e + 127)
        s = dict(case=case, x=x, codes=codes, scales=scales, bias=None, gate=None, residual=None)
        if case["bias"]:
            s["bias"] = (rand(N) * 0.1).bfloat16()
        if case["gate"]:
            rows = -(-M // 2)  # two images
            s["gate"] = ((rand(6, N) / math.sqrt(N)).bfloat16(), (rand(2, 6 * N) * 0.5).bfloat16(), 5, rows)
            s["residual"] = rand(M, N).bfloat16()
        return s
    H, Hk, D, B = case["H"], case["Hk"], case["D"], case["B"]
    N = case.get("N", 1)
    dt = _dt(case)
    qkv = rand(B * N, (H + 2 * Hk) * D).to(dt)  # column blocks of one projection
    steps = torch.arange(H, device=DEV) / max(1, H - 1)
    log_decay = -torch.exp2(-1 - 9 * steps - 0.2 * torch.rand(H, generator=g, device=DEV))  # half a token to a thousand
    s = dict(case=case, q=qkv[:, : H * D], k=qkv[:, H * D: (H + Hk) * D], v=qkv[:, (H + Hk) * D:], log_decay=log_decay,
             scale=1.0 if case["relu"] else D ** -0.5, eps=case["eps"] if case["relu"] and case["eps"] > 0 else None, lengths=None, prior=None,
             slots=None)

    def state(rows):
        st = rand(rows, H, D + 1, D)
        return st.abs() if case["relu"] else st  # key sums of ReLU features are not negative

    if case["op"] == "decay":
        if case["ragged"]:
            s["lengths"] = torch.randint(0, N + 1, (B,), generator=g, device=DEV).to(torch.int32)
        if case["prior"]:
            s["prior"] = state(B)
        return s
    rows = B + case["spare"]
    s["state"] = state(rows)
    slots = torch.randperm(rows, generator=g, device=DEV)[:B].to(torch.int32)
    if case["spare"] and B > 2:
        slots[B // 2] = -1  # a row of the batch that no sequence uses
    s["slots"] = slots
    return s


def work(case):
    if case["op"] == "fp8":
        M, K, N = case["M"], case["K"], case["N"]
        kb = -(-K // BLOCK)
        extra = 2 * N * case["bias"] + (2 * M * N + 3 * 2 * N) * case["gate"]
        return {"bytes": 2 * M * K + N * K + -(-N // BLOCK) * kb + 2 * M * N + extra, "flops": 2.0 * M * K * N}
    H, Hk, D, B, N = case["H"], case["Hk"], case["D"], case["B"], case.get("N", 1)
    e = 4 if case["dtype"] == "fp32" else 2
    share = 0.5 if case.get("ragged") else 1.0  # lengths are even between 0 and N; every output row is written
    state = 4 * B * H * (D + 1) * D
    tokens = e * B * N * D * ((H + 2 * Hk) * share + H)
    return {"bytes": tokens + state * (2 if case["op"] == "step" or case["prior"] else 1) + 4 * H, "flops": 4.0 * B * N * H * D * (D + 1) * share}


# ---- plain forms --------------------------------------------------------------------------------------------------


def _act(y, act):
    if act == "silu":
        return y / (1 + torch.exp(-y))
    if act == "gelu":
        return 0.5 * y * (1 + torch.tanh(0.7978845608028654 * (y + 0.044715 * y * y * y)))
    return y


def _plain_fp8(s):
    c = s["case"]
    M, K, N = c["M"], c["K"], c["N"]
    x = s["x"].float()
    e = _exponent(_blocks(x, 1)).repeat_interleave(BLOCK, 1)[:, :K]
    xq = torch.ldexp(torch.ldexp(x, -e).to(torch.float8_e4m3fn).float(), e)
    we = s["scales"].to(torch.int32).repeat_interleave(BLOCK, 0)[:N].repeat_interleave(BLOCK, 1)[:, :K] - 127
    y = xq @ torch.ldexp(s["codes"].float(), we).T
    if s["bias"] is not None:
        y = y + s["bias"].float()
    y = _act(y, c["act"])
    if s["gate"] is not None:
        table, t, row, rows = s["gate"]
        g = table[row].float() + t.reshape(2, 6, N)[:, row].float()
        y = y * g.repeat_interleave(rows, 0)[:M] + s["residual"].float()
    return y.bfloat16()


def _heads(t, B, N, heads, D, H):
    """[B*N, heads*D] -> fp32 [B, H, N, D]; key/value heads are shared by neighbouring query heads."""
    return t.float().reshape(B, N, heads, D).transpose(1, 2).repeat_interleave(H // heads, 1)


def _plain_decay(s):
    c = s["case"]
    B, N, H, Hk, D, C = c["B"], c["N"], c["H"], c["Hk"], c["D"], 128
    q, k, v = _heads(s["q"], B, N, H, D, H), _heads(s["k"], B, N, Hk, D, H), _heads(s["v"], B, N, Hk, D, H)
    if c["relu"]:
        q, k = q.clamp(min=0), k.clamp(min=0)
    pos = torch.arange(N, device=q.device)
    length = s["lengths"].long() if s["lengths"] is not None else torch.full((B,), N, device=q.device)
    live = (pos < length[:, None])[:, None, :, None]
    v = torch.cat([v, torch.ones_like(v[..., :1])], -1) * live
    k = k * live
    g = s["log_decay"]
    nc = -(-N // C)

    def chunks(t):
        return torch.nn.functional.pad(t, (0, 0, 0, nc * C - N)).reshape(B, H, nc, C, t.shape[-1])

    qc, kc, vc = chunks(q), chunks(k), chunks(v)
    i = torch.arange(C, device=q.device)
    dist = i[:, None] - i
    mask = torch.where(dist >= 0, torch.exp(g[:, None, None] * dist.clamp(min=0)), 0.0)  # [H, C, C]
    intra = (qc @ kc.transpose(-1, -2) * mask[:, None]) @ vc
    part = (vc * torch.exp(g[:, None] * (C - 1 - i))[:, None, :, None]).transpose(-1, -2) @ kc  # [B, H, nc, D+1, D]
    cc = torch.arange(nc, device=q.device)
    far = cc[:, None] - 1 - cc
    link = torch.where(far >= 0, torch.exp(g[:, None, None] * (C * far.clamp(min=0))), 0.0)
    before = (link @ part.reshape(B, H, nc, -1)).reshape(part.shape)
    if s["prior"] is not None:
        before = before + torch.exp(g[:, None] * (C * cc))[:, :, None, None] * s["prior"][:, :, None]
    inter = (qc * torch.exp(g[:, None] * (i + 1))[:, None, :, None]) @ before.transpose(-1, -2)
    o = (intra + inter).reshape(B, H, nc * C, D + 1)[:, :, :N]
    if s["eps"] is not None:
        o = o[..., :D] / (o[..., D:] + s["eps"])
    else:
        o = o[..., :D] * s["scale"]
    o = (o * live).transpose(1, 2).reshape(B * N, H * D).to(_dt(c))
    left = (length[:, None] - 1 - pos).clamp(min=0)
    state = (v * torch.exp(g[:, None] * left[:, None])[..., None]).transpose(-1, -2) @ k
    if s["prior"] is not None:
        state = state + torch.exp(g * length[:, None])[..., None, None] * s["prior"]
    return o, state


def _plain_step(s):
    c = s["case"]
    B, H, Hk, D = c["B"], c["H"], c["Hk"], c["D"]
    q, k, v = (_heads(s[n], B, 1, h, D, H)[:, :, 0] for n, h in (("q", H), ("k", Hk), ("v", Hk)))
    if c["relu"]:
        q, k = q.clamp(min=0), k.clamp(min=0)
    used = s["slots"] >= 0
    at = s["slots"].long().clamp(min=0)
    old = s["state"][at]
    v1 = torch.cat([v, torch.ones_like(v[..., :1])], -1)
    new = old * torch.exp(s["log_decay"])[:, None, None] + v1[..., None] * k[..., None, :]
    o = (new * q[..., None, :]).sum(-1)
    o = o[..., :D] / (o[..., D:] + s["eps"]) if s["eps"] is not None else o[..., :D] * s["scale"]
    s["state"].index_add_(0, at, (new - old) * used[:, None, None, None])  # nothing for an unused row
    return (o * used[:, None, None]).reshape(B, H * D).to(_dt(c)), s["state"]


def run(state):
    s, c = state, state["case"]
    if not own:
        return {"fp8": _plain_fp8, "decay": _plain_decay, "step": _plain_step}[c["op"]](s)
    from sana_b200 import ops
    if c["op"] == "fp8":
        act = {"none": ops.ACT_NONE, "silu": ops.ACT_SILU, "gelu": ops.ACT_GELU_TANH}[c["act"]]
        w = ops.Fp8Tensor(s["codes"], s["scales"], block_rows=BLOCK)
        return ops.gemm_fp8(ops.fp8_quantize(s["x"]), w, bias=s["bias"], act=act, gate=s["gate"], residual=s["residual"])
    if c["op"] == "decay":
        return ops.la_decay(s["q"], s["k"], s["v"], s["log_decay"], c["B"], c["N"], c["H"], c["D"], scale=s["scale"],
                            relu=c["relu"], eps=s["eps"], prior=s["prior"], lengths=s["lengths"])
    o = ops.la_decay_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"], c["H"], c["D"], scale=s["scale"],
                          relu=c["relu"], eps=s["eps"], slots=s["slots"])
    return o, s["state"]


# ---- 64-bit values ------------------------------------------------------------------------------------------------


def _exact_fp8(s):
    c = s["case"]
    M, K, N = c["M"], c["K"], c["N"]
    x = s["x"].double()
    xq = torch.empty_like(x)
    w = torch.empty(N, K, dtype=torch.float64, device=x.device)
    for b, k0 in enumerate(range(0, K, BLOCK)):
        part = x[:, k0:k0 + BLOCK]
        amax = part.abs().amax(1, keepdim=True)
        unit = torch.exp2(torch.ceil(torch.log2(amax.clamp(min=2.0 ** -126) / 448)).clamp(min=-126))
        unit = torch.where(amax > 448 * unit, 2 * unit, unit)  # log2 next to a power of two
        unit = torch.where((amax <= 224 * unit) & (unit > 2.0 ** -126), unit / 2, unit)
        xq[:, k0:k0 + BLOCK] = (part / unit).float().to(torch.float8_e4m3fn).double() * unit
        units = torch.exp2(s["scales"][:, b].double() - 127).repeat_interleave(BLOCK)[:N, None]
        w[:, k0:k0 + BLOCK] = s["codes"][:, k0:k0 + BLOCK].double() * units
    y = torch.empty(M, N, dtype=torch.float64, device=x.device)
    for m0 in range(0, M, 4096):
        z = xq[m0:m0 + 4096] @ w.T
        if s["bias"] is not None:
            z += s["bias"].double()
        if c["act"] == "silu":
            z = z * torch.sigmoid(z)
        elif c["act"] == "gelu":
            z = torch.nn.functional.gelu(z, approximate="tanh")
        if s["gate"] is not None:
            table, t, row, rows = s["gate"]
            image = torch.arange(m0, min(M, m0 + 4096), device=x.device) // rows
            z = z * (table[row].double() + t.double()[image, row * N:(row + 1) * N]) + s["residual"][m0:m0 + 4096].double()
        y[m0:m0 + 4096] = z
    return y


def _exact_decay(s):
    """Every output from the sum over all earlier tokens, one head of one sequence and 2 048 rows at a time."""
    c = s["case"]
    B, N, H, Hk, D = c["B"], c["N"], c["H"], c["Hk"], c["D"]
    out = torch.zeros(B, N, H, D, dtype=torch.float64, device=DEV)
    state = torch.zeros(B, H, D + 1, D, dtype=torch.float64, device=DEV)
    ends = s["lengths"].tolist() if s["lengths"] is not None else [N] * B
    g = s["log_decay"].double().tolist()
    phi = torch.relu if c["relu"] else (lambda t: t)
    for b in range(B):
        n = ends[b]
        rows = slice(b * N, b * N + n)
        for h in range(H):
            kv = h // (H // Hk)
            q = phi(s["q"][rows, h * D:(h + 1) * D].double())
            k = phi(s["k"][rows, kv * D:(kv + 1) * D].double())
            v = torch.ones(n, D + 1, dtype=torch.float64, device=DEV)
            v[:, :D] = s["v"][rows, kv * D:(kv + 1) * D].double()
            t = torch.arange(n, device=DEV, dtype=torch.float64)
            start = s["prior"][b, h].double() if s["prior"] is not None else None
            for n0 in range(0, n, 2048):
                n1 = min(n, n0 + 2048)
                d = t[n0:n1, None] - t[None, :n1]
                a = q[n0:n1] @ k[:n1].T * torch.exp(g[h] * d.clamp(min=0)) * (d >= 0)
                o = a @ v[:n1]
                if start is not None:
                    o += torch.exp(g[h] * (t[n0:n1, None] + 1)) * (q[n0:n1] @ start.T)
                out[b, n0:n1, h] = o[:, :D] / (o[:, D:] + s["eps"]) if s["eps"] is not None else o[:, :D] * s["scale"]
            state[b, h] = (v * torch.exp(g[h] * (n - 1 - t))[:, None]).T @ k
            if start is not None:
                state[b, h] += math.exp(g[h] * n) * start
    return out.reshape(B * N, H * D), state


def _exact_step(s):
    c = s["case"]
    B, H, Hk, D = c["B"], c["H"], c["Hk"], c["D"]
    out = torch.zeros(B, H, D, dtype=torch.float64, device=DEV)
    state = s["state"].double()
    lam = torch.exp(s["log_decay"].double())[:, None, None]
    phi = torch.relu if c["relu"] else (lambda t: t)
    head = torch.arange(H, device=DEV) // (H // Hk)
    for b, slot in enumerate(s["slots"].tolist()):
        if slot < 0:
            continue
        q = phi(s["q"][b].double().reshape(H, D))
        k = phi(s["k"][b].double().reshape(Hk, D))[head]
        v = s["v"][b].double().reshape(Hk, D)[head]
        state[slot] *= lam
        state[slot, :, :D] += torch.einsum("hi,hj->hij", v, k)
        state[slot, :, D] += k
        o = torch.einsum("hij,hj->hi", state[slot], q)
        out[b] = o[:, :D] / (o[:, D:] + s["eps"]) if s["eps"] is not None else o[:, :D] * s["scale"]
    return out.reshape(B, H * D), state


def exact(case, seed):
    s = prepare(case, seed)
    return {"fp8": _exact_fp8, "decay": _exact_decay, "step": _exact_step}[case["op"]](s)
