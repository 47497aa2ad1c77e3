"""Cases of the FP8-block product, cross attention and gated residual norm, with their plain forms.

Layout of one case: ``kind`` is ``cast`` (activation cast to E4M3 codes with a scale per 1 x 128 block),
``linear`` (that cast and the product with a weight held as E4M3 codes with a scale per 128 x 128 block),
``cross`` (attention of queries over keys of another length) or ``norm`` (post-norm, gate, residual scale,
residual add, pre-norm, optionally cast to the FP8 block format).
"""
import math
import os
import sys

import torch

own = False

DT = {"bf16": torch.bfloat16, "f32": torch.float32}
F8 = torch.float8_e4m3fn


def _api():
    """The framework's package (its folder is not importable by name: it holds a hyphen)."""
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vit-nvfp4_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from vitfp4 import nvfp4
    return nvfp4


# --------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # activations of one ViT-L/14 image on their way into an FP8 layer
        {"name": "cast image", "kind": "cast", "m": 257, "k": 1024, "dtype": "bf16"},
        # MLP hidden activations of a batch of ViT-H/14 images at 448 pixels
        {"name": "cast hidden batch", "kind": "cast", "m": 16400, "k": 5120, "dtype": "bf16"},
        # one token through a ViT-L sized fc1: a decoder's step, or a class token's head
        {"name": "linear token", "kind": "linear", "m": 1, "n": 4096, "k": 1024, "bias": True, "dtype": "bf16"},
        # one image through the same layer
        {"name": "linear image", "kind": "linear", "m": 257, "n": 4096, "k": 1024, "bias": True, "dtype": "bf16"},
        # a 1000-class head over pooled features, a width that is no multiple of 128
        {"name": "linear head ragged", "kind": "linear", "m": 512, "n": 1000, "k": 1176, "bias": True, "dtype": "bf16"},
        # fc1 of ViT-H/14 over a batch of 448-pixel images
        {"name": "linear batch", "kind": "linear", "m": 16400, "n": 5120, "k": 1280, "bias": True, "dtype": "bf16"},
        # attention pooling: one latent query per image over a ViT-L/14 encoder's 257 tokens
        {"name": "cross pool", "kind": "cross", "b": 64, "h": 16, "hkv": 16, "sq": 1, "skv": 257, "d": 64, "mask": "none"},
        # one decoder token over a long encoder memory (video, many tiles), shared KV heads, ragged lengths
        {"name": "cross token long", "kind": "cross", "b": 4, "h": 32, "hkv": 8, "sq": 1, "skv": 16391, "d": 128, "mask": "lens"},
        # 64 latents over the 1025 tokens of ViT-H/14 at 448 pixels, images of several sizes in the batch
        {"name": "cross latents", "kind": "cross", "b": 32, "h": 16, "hkv": 16, "sq": 64, "skv": 1025, "d": 80, "mask": "lens"},
        # decoder tokens over four images' tokens with dropped patches
        {"name": "cross decoder", "kind": "cross", "b": 8, "h": 16, "hkv": 16, "sq": 1030, "skv": 4100, "d": 64, "mask": "keys"},
        # sandwich norms of one ViT-L image, the FP8 operand of the next layer written
        {"name": "norm image", "kind": "norm", "m": 257, "k": 1024, "groups": 1, "norm": "layer", "affine": True, "out": "fp8", "dtype": "bf16"},
        # the same over a batch, a gate per image
        {"name": "norm batch", "kind": "norm", "m": 65792, "k": 1024, "groups": 256, "norm": "rms", "affine": True, "out": "same", "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["cast", "linear", "cross", "norm"])
    if kind == "cast":
        k = _log(rng, 64, 8192)
        return {"kind": kind, "m": _log(rng, 1, min(65536, 16400 * 5120 // k)), "k": k, "dtype": rng.choice(["bf16", "f32"])}
    if kind == "linear":
        n, k = _log(rng, 48, 5120), _log(rng, 48, 5120)
        return {"kind": kind, "m": _log(rng, 1, min(16400, 16400 * 5120 * 1280 // (n * k))), "n": n, "k": k,
                "bias": rng.random() < 0.5, "dtype": "bf16"}
    if kind == "cross":
        d, hkv, group = rng.choice([32, 64, 72, 80, 96, 128]), rng.choice([1, 2, 4, 8, 12, 16]), rng.choice([1, 1, 2, 4])
        sq, skv = _log(rng, 1, 2048), _log(rng, 1, 32768)
        one = hkv * (group * sq * skv * 2.0 + (skv + group * sq) * d * 8.0)   # scores, and the operands themselves
        room = 8 * 16 * 1030 * 4100 * 2.0 * min(1.0, 64 / d)
        most = int(room // one)
        if most < 1:
            skv = max(1, int(skv * room / one))
        return {"kind": kind, "b": _log(rng, 1, max(1, min(128, most))), "h": hkv * group, "hkv": hkv, "sq": sq, "skv": skv,
                "d": d, "mask": rng.choice(["none", "lens", "keys"])}
    k, groups = _log(rng, 64, 8192), rng.choice([1, 1, 3, 16])
    rows = _log(rng, 1, max(1, min(65792, 65792 * 1024 // (2 * k)) // groups))
    return {"kind": kind, "m": rows * groups, "k": k, "groups": groups, "norm": rng.choice(["layer", "rms"]),
            "affine": rng.random() < 0.8, "out": rng.choice(["same", "fp8"]), "dtype": rng.choice(["bf16", "f32"])}


# -------------------------------------------------------------------------------------------- inputs
def _rows(k):
    """Row length of E4M3 codes in memory: rows begin on 16-byte boundaries."""
    return (k + 15) // 16 * 16


def _activations(m, k, g, dtype):
    """N(0, 1) with a few channels 20 times as large, as the hidden states of a trained ViT have them."""
    x = torch.randn(m, k, generator=g, device="cuda")
    heavy = torch.randperm(k, generator=g, device="cuda")[: max(1, k // 1000)]
    x[:, heavy] *= 20
    return x.to(dtype)


def _weight(n, k, g):
    """An FP8 checkpoint's weight: codes (n, k) in rows padded to 16 bytes, scales (n / 128, k / 128)."""
    w = torch.randn(n, k, generator=g, device="cuda") * 0.02
    nb, kb = -(-n // 128), -(-k // 128)
    full = torch.zeros(nb * 128, kb * 128, device="cuda")
    full[:n, :k] = w
    blocks = full.view(nb, 128, kb, 128)
    amax = blocks.abs().amax(dim=(1, 3)).clamp(min=1e-12)
    scale = amax / 448.0
    codes = (blocks * 448.0 / amax[:, None, :, None]).clamp(-448, 448).reshape(nb * 128, kb * 128)[:n, :k]
    buf = torch.zeros(n, _rows(k), device="cuda").to(F8)
    buf[:, :k] = codes.to(F8)
    return buf[:, :k], scale.contiguous()


def _lens(b, skv):
    """Key counts of a ragged batch: spread over the range, the first whole, one image in eight without keys."""
    return [0 if i % 8 == 5 else max(1, int(skv * (1 - (i * 0.381966) % 1.0 * 0.75))) for i in range(b)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = dict(case)
    if c["kind"] == "cast":
        c["x"] = _activations(c["m"], c["k"], g, DT[c["dtype"]])
    elif c["kind"] == "linear":
        c["x"] = _activations(c["m"], c["k"], g, DT[c["dtype"]])
        c["w"], c["ws"] = _weight(c["n"], c["k"], g)
        c["b"] = torch.randn(c["n"], generator=g, device="cuda").bfloat16() if c["bias"] else None
    elif c["kind"] == "cross":
        # (B, H, S, D) views of the projections' (B, S, H * D) outputs; K and V of one projection of the encoder's states
        q = torch.randn(c["b"], c["sq"], c["h"], c["d"], generator=g, device="cuda").bfloat16()
        kv = torch.randn(c["b"], c["skv"], 2, c["hkv"], c["d"], generator=g, device="cuda", dtype=torch.float32).bfloat16()
        c["q"], c["kk"], c["v"] = q.transpose(1, 2), kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
        c["lens"] = c["keep"] = None
        if c["mask"] == "lens":
            c["lens"] = torch.tensor(_lens(c["b"], c["skv"]), dtype=torch.int32, device="cuda")
        elif c["mask"] == "keys":
            c["keep"] = torch.rand(c["b"], c["skv"], generator=g, device="cuda") < 0.75
    else:
        dt, k = DT[c["dtype"]], c["k"]
        c["x"] = _activations(c["m"], k, g, dt)
        c["y"] = torch.randn(c["m"], k, generator=g, device="cuda").to(dt)
        c["gate"] = torch.randn(*((c["groups"], k) if c["groups"] > 1 else (k,)), generator=g, device="cuda").to(dt)
        aff = lambda base: (base + 0.1 * torch.randn(k, generator=g, device="cuda")).to(dt)
        c["w2"], c["w1"] = (aff(1.0), aff(1.0)) if c["affine"] else (None, None)
        c["b2"], c["b1"] = (aff(0.0), aff(0.0)) if c["affine"] and c["norm"] == "layer" else (None, None)
    return c


# ----------------------------------------------------------------------------------------- plain forms
def _plain_cast(x):
    m, k = x.shape
    kb = -(-k // 128)
    xf = torch.nn.functional.pad(x.float(), (0, kb * 128 - k)).view(m, kb, 128)
    amax = xf.abs().amax(dim=2).clamp(min=1e-12)
    codes = (xf * 448.0 / amax[:, :, None]).clamp(-448, 448).to(F8).view(m, kb * 128)[:, :k]
    return codes, amax / 448.0


def _plain_norm(x, kind, w, b):
    if kind == "layer":
        x = x - x.mean(dim=1, keepdim=True)
    x = x * torch.rsqrt((x * x).mean(dim=1, keepdim=True) + 1e-6)
    if w is not None:
        x = x * w.float()
    return x if b is None else x + b.float()


def _plain(c):
    if c["kind"] == "cast":
        return _plain_cast(c["x"])
    if c["kind"] == "linear":
        codes, scale = _plain_cast(c["x"])
        n, k = c["w"].shape
        a = codes.float() * scale.repeat_interleave(128, dim=1)[:, :k]
        w = c["w"].float() * c["ws"].repeat_interleave(128, dim=0)[:n].repeat_interleave(128, dim=1)[:, :k]
        y = a @ w.t()
        if c["b"] is not None:
            y = y + c["b"].float()
        return y.to(c["x"].dtype)
    if c["kind"] == "cross":
        b, h, sq, d = c["q"].shape
        hkv, skv = c["kk"].shape[1], c["kk"].shape[2]
        q = c["q"].float().reshape(b, hkv, h // hkv * sq, d)
        s = (q * d ** -0.5) @ c["kk"].float().transpose(2, 3)
        keep = c["keep"]
        if c["lens"] is not None:
            keep = torch.arange(skv, device="cuda")[None, :] < c["lens"][:, None]
        if keep is not None:
            s = s.masked_fill(~keep[:, None, None, :], -torch.inf)
        top = s.amax(dim=3, keepdim=True)
        p = torch.exp(s - torch.where(torch.isfinite(top), top, 0.0))
        total = p.sum(dim=3, keepdim=True)
        o = (p @ c["v"].float()) / torch.where(total > 0, total, 1.0)
        return o.view(b, h, sq, d).bfloat16()
    x, y = c["x"].float(), c["y"].float()
    gate = c["gate"].float().view(-1, c["k"]).repeat_interleave(c["m"] // c["groups"], dim=0)
    new = x + 0.5 * gate * _plain_norm(y, c["norm"], c["w2"], c["b2"])
    nxt = _plain_norm(new, c["norm"], c["w1"], c["b1"])
    return new.to(c["x"].dtype), (_plain_cast(nxt) if c["out"] == "fp8" else nxt.to(c["x"].dtype))


def run(state):
    c = state
    if not own:
        return _plain(c)
    api = _api()
    if c["kind"] == "cast":
        return api.quantize_to_fp8_block(c["x"])
    if c["kind"] == "linear":
        return api.fp8_block_linear(c["x"], c["w"], c["ws"], bias=c["b"])
    if c["kind"] == "cross":
        return api.cross_sdpa(c["q"], c["kk"], c["v"], kv_lens=c["lens"], key_mask=c["keep"])
    return api.gated_residual_norm(c["x"], c["y"], gate=c["gate"], residual_scale=0.5, norm=c["norm"],
                                   post_weight=c["w2"], post_bias=c["b2"], pre_weight=c["w1"], pre_bias=c["b1"],
                                   eps=1e-6, out_dtype=F8 if c["out"] == "fp8" else None)


# ------------------------------------------------------------------------------------------ accounting
def work(case):
    c = case
    e = 2 if c.get("dtype", "bf16") == "bf16" else 4
    if c["kind"] == "cast":
        m, k = c["m"], c["k"]
        return {"bytes": m * k * (e + 1) + m * -(-k // 128) * 4, "flops": 3 * m * k}
    if c["kind"] == "linear":
        m, n, k = c["m"], c["n"], c["k"]
        return {"bytes": m * k * e + n * k + -(-n // 128) * -(-k // 128) * 4 + m * n * e + (2 * n if c["bias"] else 0),
                "flops": 2 * m * n * k}
    if c["kind"] == "cross":
        keys = sum(_lens(c["b"], c["skv"])) if c["mask"] == "lens" else c["b"] * c["skv"]
        return {"bytes": 4 * c["b"] * c["h"] * c["sq"] * c["d"] + 4 * keys * c["hkv"] * c["d"]
                + (c["b"] * c["skv"] if c["mask"] == "keys" else 4 * c["b"] if c["mask"] == "lens" else 0),
                "flops": 4 * keys * c["h"] * c["sq"] * c["d"]}
    m, k = c["m"], c["k"]
    out = k + -(-k // 128) * 4 if c["out"] == "fp8" else k * e
    return {"bytes": m * (3 * k * e + out) + (c["groups"] + 4) * k * e, "flops": 16 * m * k}


# ----------------------------------------------------------------------------------------------- exact
def _exact_blocks(x):
    """Codes and scales of float64 rows, block by block of 128 columns."""
    codes, scales = [], []
    for part in x.split(128, dim=1):
        top = part.abs().max(dim=1, keepdim=True).values
        top = torch.maximum(top, torch.full_like(top, 1e-12))
        v = part * 448.0 / top
        # nearest E4M3 value, ties to even: steps of 2^(e-3) in the binade 2^e, of 2^-9 below 2^-6
        step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
        codes.append(torch.round(v / step) * step)
        scales.append(top / 448.0)
    return torch.cat(codes, 1), torch.cat(scales, 1)


def exact(case, seed):
    c = prepare(case, seed)
    if c["kind"] == "cast":
        codes, scale = _exact_blocks(c["x"].double())
        return codes, scale
    if c["kind"] == "linear":
        codes, scale = _exact_blocks(c["x"].double())
        n, k = c["w"].shape
        w = c["w"].double()
        y = torch.zeros(c["m"], n, dtype=torch.float64, device="cuda")
        rows = torch.arange(n, device="cuda") // 128
        for g in range(-(-k // 128)):
            cut = slice(128 * g, min(k, 128 * g + 128))
            part = torch.mm(codes[:, cut], w[:, cut].t())
            y += part * scale[:, g : g + 1] * c["ws"][:, g].double()[rows][None, :]
        return y if c["b"] is None else y + c["b"].double()[None, :]
    if c["kind"] == "cross":
        b, h, sq, d = c["q"].shape
        group = h // c["hkv"]
        out = torch.zeros(b, h, sq, d, dtype=torch.float64, device="cuda")
        lens = _lens(b, c["skv"]) if c["mask"] == "lens" else [c["skv"]] * b
        for i in range(b):
            at = torch.arange(lens[i], device="cuda") if c["keep"] is None else c["keep"][i].nonzero()[:, 0]
            if at.numel() == 0:
                continue
            for j in range(c["hkv"]):
                k, v = c["kk"][i, j][at].double(), c["v"][i, j][at].double()
                for t in range(j * group, (j + 1) * group):
                    s = torch.mm(c["q"][i, t].double(), k.t()) / math.sqrt(d)
                    out[i, t] = torch.mm(torch.exp(s - torch.logsumexp(s, dim=1, keepdim=True)), v)
        return out

    def norm(t, w, bias):
        if c["norm"] == "layer":
            z = (t - t.mean(1, keepdim=True)) / torch.sqrt(t.var(1, unbiased=False, keepdim=True) + 1e-6)
        else:
            z = t / torch.sqrt(t.pow(2).mean(1, keepdim=True) + 1e-6)
        z = z if w is None else z * w.double()
        return z if bias is None else z + bias.double()

    per = c["m"] // c["groups"]
    new = c["x"].double()
    branch = norm(c["y"].double(), c["w2"], c["b2"])
    for i in range(c["groups"]):
        new[i * per : (i + 1) * per] += 0.5 * c["gate"].double().reshape(-1, c["k"])[i] * branch[i * per : (i + 1) * per]
    nxt = norm(new, c["w1"], c["b1"])
    return new, (_exact_blocks(nxt) if c["out"] == "fp8" else nxt)
