"""Workloads of the group-norm and cross-attention operators: what is timed, in a plain form and through the package.

Row layout throughout: an image map is ``[B * n, C]`` (NHWC pixels), a token sequence ``[B * n, heads * hd]``.

group norm with an activation
    mean, var over the n x (C / groups) elements of a group; ``xh = (x - mean) / sqrt(var + eps)``;
    ``z = (xh * gamma + beta) * (1 + scale_b) + shift_b``; ``y = act(z)`` with act = none or SiLU.
cross attention
    ``o = softmax(scale * q k^T) v`` over the keys an image shows (a length per image and / or a mask per key), head h of
    q reading key / value head ``h // (heads / kv_heads)``; an image that shows no key gives zeros.
"""
from __future__ import annotations

import math

import torch

own = False   # True: run() calls the package's kernels; False: the plain forms below

EPS = 1e-6
DT = {"bf16": torch.bfloat16, "f32": torch.float32}
ESIZE = {"bf16": 2, "f32": 4}

# the largest work of a listed case, per kind: a drawn case stays below it
MAX_GN = 16 * 65536 * 64          # elements of a map
MAX_FWD_PAIRS = 8 * 8 * 16384 * 577   # (head, query, key) triples, forward
MAX_BWD_PAIRS = 4 * 8 * 4096 * 1152   # and backward
MAX_ROWS = 16 * 8192 * 512        # elements of any one token tensor


def _gn(name, kind, B, n, C, groups, act, ss, dt):
    return {"name": name, "kind": kind, "B": B, "n": n, "C": C, "groups": groups, "act": act, "ss": ss, "dt": dt}


def _ca(name, kind, B, nq, nk, heads, kv, hd, keys, dt):
    return {"name": name, "kind": kind, "B": B, "nq": nq, "nk": nk, "heads": heads, "kv": kv, "hd": hd, "keys": keys, "dt": dt}


def listed():
    return [
        # ---- group norm, forward
        # the bottom map of the UNet (nf = 64, mult 8) for one 64 x 64 crop: a sampling step's latency
        _gn("gn_bottom_8x8_f32", "gn_fwd", 1, 64, 512, 32, "none", False, "f32"),
        # a time-modulated residual block's norm at 64 x 64, batch 8
        _gn("gn_silu_mod_64x64", "gn_fwd", 8, 4096, 256, 32, "silu", True, "bf16"),
        # level 0 of a 256 x 256 batch of 16: the largest map a sampler norms
        _gn("gn_silu_256x256", "gn_fwd", 16, 65536, 64, 32, "silu", False, "bf16"),
        # ---- group norm, backward
        # a 19 x 22 map (even-size frames halve to it) with 3 channels a group
        _gn("gn_bwd_19x22_c96_f32", "gn_bwd", 3, 418, 96, 32, "none", False, "f32"),
        # training step of a modulated block at 128 x 128
        _gn("gn_bwd_silu_mod_128x128", "gn_bwd", 8, 16384, 128, 32, "silu", True, "bf16"),
        # full-resolution map in single precision
        _gn("gn_bwd_silu_256x256_f32", "gn_bwd", 8, 65536, 64, 32, "silu", False, "f32"),
        # ---- cross attention, forward
        # one pooling query an image over long, ragged states, four query heads to a key head
        _ca("ca_one_query_8192", "ca_fwd", 16, 1, 8192, 32, 8, 64, "lens", "bf16"),
        # a 32 x 32 map over the 50 states of a ViT-B/32 encoder, the UNet's heads of 32
        _ca("ca_32x32_vit50", "ca_fwd", 8, 1024, 50, 8, 8, 32, "none", "bf16"),
        # a 128 x 128 map over 577 states (24 x 24 patches and a class token): the largest product
        _ca("ca_128x128_states577", "ca_fwd", 8, 16384, 577, 8, 8, 64, "none", "bf16"),
        # single precision, padded caption states under a mask
        _ca("ca_32x32_masked197_f32", "ca_fwd", 2, 1024, 197, 16, 16, 32, "mask", "f32"),
        # ---- cross attention, backward
        # training step of a 64 x 64 map over padded caption states
        _ca("ca_bwd_64x64_masked77", "ca_bwd", 8, 4096, 77, 8, 8, 32, "mask", "bf16"),
        # long states with shared key heads
        _ca("ca_bwd_64x64_states2048", "ca_bwd", 4, 4096, 2048, 8, 2, 64, "lens", "bf16"),
    ]


def _log(rng, lo, hi):
    return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))


def draw(rng):
    kind = rng.choice(["gn_fwd", "gn_bwd", "ca_fwd", "ca_fwd", "ca_bwd"])
    dt = rng.choice(["bf16", "bf16", "f32"])
    B = rng.randint(1, 16)
    if kind.startswith("gn"):
        groups = rng.choice([1, 4, 8, 16, 32, 32])
        C = groups * rng.randint(1, 1024 // groups if groups < 8 else 24)
        top = MAX_GN if kind == "gn_fwd" and dt == "bf16" else MAX_GN // 2 - 65536
        n = _log(rng, 1, 65536)
        n = max(1, min(n, top // (B * C)))
        c = _gn("", kind, B, n, C, groups, rng.choice(["none", "silu"]), rng.random() < 0.5, dt)
    else:
        hd = rng.choice([16, 24, 32, 40, 64, 64, 80, 96, 128])
        kv = rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([1, 1, 2, 4])
        heads = heads if heads <= 16 else kv
        nq = 1 if rng.random() < 0.25 else _log(rng, 1, 16384)
        nk = _log(rng, 1, 8192)
        # products of 2 * hd flops a triple: wide heads take fewer triples; single precision has a sixteenth of the rate
        top = (MAX_FWD_PAIRS if kind == "ca_fwd" else MAX_BWD_PAIRS) * 64 // max(64, hd)
        if dt == "f32":
            top //= 8
        rows = MAX_ROWS // ((1 if dt == "bf16" else 2) * (1 if kind == "ca_fwd" else 2))
        nk = max(1, min(nk, rows // (B * kv * hd)))
        nq = max(1, min(nq, top // (B * heads * nk), rows // (B * heads * hd)))
        c = _ca("", kind, B, nq, nk, heads, kv, hd, rng.choice(["none", "lens", "mask", "both"]), dt)
    del c["name"]
    return c


def _visible(case):
    """Keys an image shows by its length, in some order over the images: known from the case, shuffled by the seed."""
    B, nk = case["B"], case["nk"]
    if case["keys"] not in ("lens", "both"):
        return [nk] * B
    lens = [(nk * (i + 1) + B - 1) // B for i in range(B)]
    if B >= 4:
        lens[0] = 0   # an image whose condition was dropped
    return lens


def work(case):
    es = ESIZE[case["dt"]]
    B = case["B"]
    if case["kind"].startswith("gn"):
        e, C = B * case["n"] * case["C"], case["C"]
        small = 4 * (2 * C + (2 * B * C if case["ss"] else 0))
        if case["kind"] == "gn_fwd":
            return {"bytes": 2 * e * es + small, "flops": 8 * e}
        return {"bytes": 3 * e * es + 2 * small + 8 * B * case["groups"], "flops": 20 * e}
    rows = sum(_visible(case))
    qe = B * case["nq"] * case["heads"] * case["hd"]
    kve = rows * case["kv"] * case["hd"]
    full = B * case["nk"] * case["kv"] * case["hd"]
    pairs = case["heads"] * case["nq"] * rows
    aux = (B * case["nk"] if case["keys"] in ("mask", "both") else 0) + (4 * B if case["keys"] in ("lens", "both") else 0)
    if case["kind"] == "ca_fwd":
        return {"bytes": (2 * qe + 2 * kve) * es + aux, "flops": 4 * pairs * case["hd"]}
    lse = 4 * B * case["heads"] * case["nq"]
    return {"bytes": (4 * qe + 2 * kve + 2 * full) * es + aux + lse, "flops": 10 * pairs * case["hd"]}


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DT[case["dt"]]
    B = case["B"]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    st = {"case": case}
    if case["kind"].startswith("gn"):
        n, C, G = case["n"], case["C"], case["groups"]
        # feature maps: every channel has an offset and a spread of its own
        x = randn(B * n, C) * (0.5 + randn(C).abs()) + randn(C)
        st["x"] = x.to(dt)
        st["gamma"], st["beta"] = 1.0 + 0.2 * randn(C), 0.2 * randn(C)
        st["ss"] = 0.3 * randn(B, 2 * C) if case["ss"] else None
        if case["kind"] == "gn_bwd":
            st["dy"] = randn(B * n, C).to(dt)
            xg = st["x"].view(B, n, G, C // G)   # what the forward pass kept
            means, rstds = [], []
            for b in range(B):
                xb = xg[b].double()
                m = xb.mean((0, 2))
                v = (xb - m[None, :, None]).square().mean((0, 2))
                means.append(m)
                rstds.append((v + EPS).rsqrt())
            st["mean"], st["rstd"] = torch.stack(means).float(), torch.stack(rstds).float()
        if own:
            from underwater_image_restoration_amd import ops
            st["ws"] = torch.empty(max(ops.group_norm_act_workspace_bytes(B, n, C, G), 16), dtype=torch.uint8, device=dev)
            st["out"] = torch.empty(B * n, C, dtype=dt, device=dev)
            if case["kind"] == "gn_bwd":
                st["dgamma"], st["dbeta"] = torch.empty(C, device=dev), torch.empty(C, device=dev)
                st["dss"] = torch.empty(B, 2 * C, device=dev) if case["ss"] else None
        return st

    nq, nk, H, KV, hd = case["nq"], case["nk"], case["heads"], case["kv"], case["hd"]
    st["q"] = (1.5 * randn(B * nq, H * hd)).to(dt)
    kvt = randn(B * nk, 2 * KV * hd).to(dt)   # one projection of the states: [k | v]
    st["k"], st["v"] = kvt[:, :KV * hd], kvt[:, KV * hd:]
    st["scale"] = 1.0 / math.sqrt(hd)
    st["lens"] = st["mask"] = None
    if case["keys"] in ("lens", "both"):
        lens = torch.tensor(_visible(case), dtype=torch.int32, device=dev)
        st["lens"] = lens[torch.randperm(B, generator=g, device=dev)]
    if case["keys"] in ("mask", "both"):
        m = torch.rand(B, nk, generator=g, device=dev) < 0.8
        if B > 1:
            m[-1, nk // 3:] = False   # a short caption in a padded batch
        st["mask"] = m
    if case["kind"] == "ca_bwd":
        st["do"] = randn(B * nq, H * hd).to(dt)
        o, lse = [], []   # what the forward pass kept
        show = _show(st)
        for b0, b1 in _chunks(case):
            p, v, m, z = _softmax(st, b0, b1, show)
            o.append(_rows(torch.matmul(p, v)))
            lse.append((m + torch.log(z)).squeeze(-1))
        st["o"], st["lse"] = torch.cat(o).to(dt), torch.cat(lse)
    if own:
        from underwater_image_restoration_amd import ops
        if case["kind"] == "ca_fwd":
            st["out"] = torch.empty(B * nq, H * hd, dtype=dt, device=dev)
            nb = ops.cross_attn_workspace_bytes(B, nq, nk, H, KV, hd, dt)
        else:
            st["dq"] = torch.empty(B * nq, H * hd, dtype=dt, device=dev)
            st["dk"], st["dv"] = torch.empty(2, B * nk, KV * hd, dtype=dt, device=dev)
            nb = ops.cross_attn_backward_workspace_bytes(B, nq, nk, H, KV, hd, dt)
        st["ws"] = torch.empty(max(nb, 16), dtype=torch.uint8, device=dev)
    return st


# ---------------------------------------------------------------------------------------------- plain forms
def _show(st):
    """[B, nk] truth values: the keys an image shows (None: all)."""
    c, show = st["case"], st["mask"]
    if st["lens"] is not None:
        inside = torch.arange(c["nk"], device="cuda")[None, :] < st["lens"][:, None]
        show = inside if show is None else show & inside
    return show


def _chunks(c):
    """images taken at a time: one product over all of them unless their scores pass 2 GiB"""
    step = max(1, 2 ** 29 // (c["heads"] * c["nq"] * c["nk"]))
    return [(b, min(c["B"], b + step)) for b in range(0, c["B"], step)]


def _heads(t, b0, b1, n, heads, hd, group=1):
    """rows of images b0..b1 as [images, heads * group, n, hd] in 32 bits, each head repeated for the queries' heads that
    share it"""
    r = t[b0 * n:b1 * n].float().view(b1 - b0, n, heads, hd).transpose(1, 2)
    if group > 1:
        r = r[:, :, None].expand(b1 - b0, heads, group, n, hd).reshape(b1 - b0, heads * group, n, hd)
    return r.contiguous()


def _softmax(st, b0, b1, show):
    """-> (probabilities of the images' keys, values, row maxima, row sums); a row that shows nothing has p = 0"""
    c = st["case"]
    H, KV, hd = c["heads"], c["kv"], c["hd"]
    q = _heads(st["q"], b0, b1, c["nq"], H, hd)
    k = _heads(st["k"], b0, b1, c["nk"], KV, hd, H // KV)
    v = _heads(st["v"], b0, b1, c["nk"], KV, hd, H // KV)
    s = torch.matmul(q, k.transpose(2, 3).contiguous()) * st["scale"]
    if show is not None:
        s = s.masked_fill(~show[b0:b1, None, None, :], float("-inf"))
    m = s.amax(-1, keepdim=True).clamp_min(-1e30)
    e = torch.exp(s - m)
    z = e.sum(-1, keepdim=True)
    return e / z.clamp_min(1e-30), v, m, z


def _rows(t):
    return t.transpose(1, 2).reshape(t.shape[0] * t.shape[2], t.shape[1] * t.shape[3])


def _plain_gn(st):
    c = st["case"]
    B, n, C, G = c["B"], c["n"], c["C"], c["groups"]
    x = st["x"].float().view(B, n, G, C // G)
    if c["kind"] == "gn_fwd":
        mean = x.mean((1, 3), keepdim=True)
        var = (x - mean).square().mean((1, 3), keepdim=True)
        xh = (x - mean) * torch.rsqrt(var + EPS)
    else:
        xh = (x - st["mean"].view(B, 1, G, 1)) * st["rstd"].view(B, 1, G, 1)
    xh = xh.view(B, n, C)
    one = torch.ones(B, 1, C, device="cuda") if st["ss"] is None else 1.0 + st["ss"][:, None, :C]
    z = (xh * st["gamma"] + st["beta"]) * one
    if st["ss"] is not None:
        z = z + st["ss"][:, None, C:]
    if c["kind"] == "gn_fwd":
        y = z / (1.0 + torch.exp(-z)) if c["act"] == "silu" else z
        return y.reshape(B * n, C).to(st["x"].dtype)
    dz = st["dy"].float().view(B, n, C)
    if c["act"] == "silu":
        sg = 1.0 / (1.0 + torch.exp(-z))
        dz = dz * (sg * (1.0 + z * (1.0 - sg)))
    s1, s2 = dz.sum(1), (dz * xh).sum(1)
    w = st["gamma"] * one
    dxh = (dz * w).view(B, n, G, C // G)
    m1 = dxh.mean((1, 3), keepdim=True)
    m2 = (dxh * xh.view(B, n, G, C // G)).mean((1, 3), keepdim=True)
    dx = (dxh - m1 - xh.view(B, n, G, C // G) * m2) * st["rstd"].view(B, 1, G, 1)
    out = [dx.reshape(B * n, C).to(st["x"].dtype), (one[:, 0] * s2).sum(0), (one[:, 0] * s1).sum(0)]
    if st["ss"] is not None:
        out.append(torch.cat([st["gamma"] * s2 + st["beta"] * s1, s1], 1))
    return out


def _plain_ca(st):
    c = st["case"]
    nq, nk, H, KV, hd = c["nq"], c["nk"], c["heads"], c["kv"], c["hd"]
    show = _show(st)
    outs = []
    for b0, b1 in _chunks(c):
        p, v, _, _ = _softmax(st, b0, b1, show)
        if c["kind"] == "ca_fwd":
            outs.append((_rows(torch.matmul(p, v)),))
            continue
        do = _heads(st["do"], b0, b1, nq, H, hd)
        dv = torch.matmul(p.transpose(2, 3).contiguous(), do)
        dp = torch.matmul(do, v.transpose(2, 3).contiguous())
        ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * st["scale"]
        dq = torch.matmul(ds, _heads(st["k"], b0, b1, nk, KV, hd, H // KV))
        dk = torch.matmul(ds.transpose(2, 3).contiguous(), _heads(st["q"], b0, b1, nq, H, hd))
        dk, dv = dk.view(-1, KV, H // KV, nk, hd).sum(2), dv.view(-1, KV, H // KV, nk, hd).sum(2)
        outs.append((_rows(dq), _rows(dk), _rows(dv)))
    outs = [torch.cat(t).to(st["q"].dtype) for t in zip(*outs)]
    return outs[0] if c["kind"] == "ca_fwd" else outs


# ---------------------------------------------------------------------------------------------- one pass
def run(st):
    c = st["case"]
    if not own:
        return _plain_gn(st) if c["kind"].startswith("gn") else _plain_ca(st)
    from underwater_image_restoration_amd import ops
    if c["kind"].startswith("gn"):
        B, n, C, G = c["B"], c["n"], c["C"], c["groups"]
        act = ops.ACT_SILU if c["act"] == "silu" else ops.ACT_NONE
        if c["kind"] == "gn_fwd":
            ops.group_norm_act(st["x"], B, n, C, G, EPS, st["gamma"], st["beta"], st["out"], st["ws"], act=act,
                               scale_shift=st["ss"])
            return st["out"]
        ops.group_norm_act_backward(st["dy"], st["x"], B, n, C, G, st["gamma"], st["beta"], st["mean"], st["rstd"], st["out"],
                                    st["dgamma"], st["dbeta"], st["ws"], act=act, scale_shift=st["ss"],
                                    dscale_shift=st["dss"])
        return [st["out"], st["dgamma"], st["dbeta"]] + ([] if st["dss"] is None else [st["dss"]])
    dims = (c["B"], c["nq"], c["nk"], c["heads"], c["kv"], c["hd"], st["scale"])
    if c["kind"] == "ca_fwd":
        ops.cross_attn(st["q"], st["k"], st["v"], *dims, st["out"], st["ws"], key_lens=st["lens"], key_mask=st["mask"])
        return st["out"]
    ops.cross_attn_backward(st["q"], st["k"], st["v"], st["o"], st["lse"], st["do"], *dims, st["dq"], st["dk"], st["dv"],
                            st["ws"], key_lens=st["lens"], key_mask=st["mask"])
    return [st["dq"], st["dk"], st["dv"]]


# ---------------------------------------------------------------------------------------------- in 64 bits
def _exact_gn(case, st):
    B, n, C, G = case["B"], case["n"], case["C"], case["groups"]
    gamma, beta = st["gamma"].double(), st["beta"].double()
    dgamma, dbeta = torch.zeros_like(gamma), torch.zeros_like(beta)
    ys, dss = [], []
    for b in range(B):
        x = st["x"][b * n:(b + 1) * n].double()
        per = x.reshape(n, G, -1).transpose(0, 1).reshape(G, -1)
        mu = per.mean(1)
        sd = ((per - mu[:, None]) ** 2).mean(1).add(EPS).sqrt()
        mu, sd = mu.repeat_interleave(C // G), sd.repeat_interleave(C // G)
        xh = (x - mu) / sd
        a, s = gamma, beta
        if st["ss"] is not None:
            sc, sh = st["ss"][b, :C].double(), st["ss"][b, C:].double()
            a, s = gamma * (1 + sc), beta * (1 + sc) + sh
        z = xh * a + s
        if case["kind"] == "gn_fwd":
            ys.append(z * torch.sigmoid(z) if case["act"] == "silu" else z)
            continue
        dz = st["dy"][b * n:(b + 1) * n].double()
        if case["act"] == "silu":
            sg = torch.sigmoid(z)
            dz = dz * (sg + z * sg * (1 - sg))
        # the reductions of one group: subtract the projections of dz * a on 1 and on xh
        h = dz * a
        t1 = h.sum(0).reshape(G, -1).sum(1) / (n * (C // G))
        t2 = (h * xh).sum(0).reshape(G, -1).sum(1) / (n * (C // G))
        ys.append((h - t1.repeat_interleave(C // G) - xh * t2.repeat_interleave(C // G)) / sd)
        s1, s2 = dz.sum(0), (dz * xh).sum(0)
        f = 1.0 if st["ss"] is None else 1 + sc
        dgamma += f * s2
        dbeta += f * s1
        dss.append(torch.cat([gamma * s2 + beta * s1, s1]))
    y = torch.cat(ys)
    if case["kind"] == "gn_fwd":
        return y
    return [y, dgamma, dbeta] + ([torch.stack(dss)] if st["ss"] is not None else [])


def _exact_ca(case, st):
    B, nq, nk, H, KV, hd = case["B"], case["nq"], case["nk"], case["heads"], case["kv"], case["hd"]
    z = dict(dtype=torch.float64, device="cuda")
    o = torch.zeros(B, nq, H, hd, **z)
    dk, dv = torch.zeros(B, nk, KV, hd, **z), torch.zeros(B, nk, KV, hd, **z)
    q4, do4 = st["q"].view(B, nq, H, hd), None if "do" not in st else st["do"].view(B, nq, H, hd)
    lens = None if st["lens"] is None else st["lens"].tolist()
    for b in range(B):
        ids = torch.arange(nk if lens is None else lens[b], device="cuda")
        if st["mask"] is not None:
            ids = ids[st["mask"][b, :len(ids)]]
        if len(ids) == 0:
            continue   # nothing is shown: zeros, and no gradient
        for h in range(H):
            j = h // (H // KV)
            kk = st["k"][b * nk + ids, j * hd:(j + 1) * hd].double()
            vv = st["v"][b * nk + ids, j * hd:(j + 1) * hd].double()
            qq = q4[b, :, h].double()
            p = torch.softmax(st["scale"] * (qq @ kk.t()), 1)
            if case["kind"] == "ca_fwd":
                o[b, :, h] = p @ vv
                continue
            g = do4[b, :, h].double()
            dp = g @ vv.t()
            ds = st["scale"] * p * (dp - (dp * p).sum(1, keepdim=True))
            o[b, :, h] = ds @ kk
            dk[b, :, j].index_add_(0, ids, ds.t() @ qq)
            dv[b, :, j].index_add_(0, ids, p.t() @ g)
    if case["kind"] == "ca_fwd":
        return o.view(B * nq, H * hd)
    return [o.view(B * nq, H * hd), dk.view(B * nk, KV * hd), dv.view(B * nk, KV * hd)]


def exact(case, seed):
    st = prepare(case, seed)
    return _exact_gn(case, st) if case["kind"].startswith("gn") else _exact_ca(case, st)
