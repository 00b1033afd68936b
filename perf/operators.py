"""Operators around a served or trained KDA layer, as measurable cases.

* ``norm``: the RMSNorm that enters a layer, with the residual's addition:
  ``fused.add_rmsnorm`` forward and backward (training), and
  ``fused.add_rmsnorm_quant`` with e4m3 output and scales (serving).
* ``adapters``: ``adapters.adapter_linear``, one shared projection of a batch
  whose requests each have a low-rank adapter of their own or none.
* ``store`` / ``load`` / ``resume``: the state cache in 8 bits.  ``cache.pack_states``
  writes the decode caches of a model's layers into slots of a pool,
  ``cache.unpack_states`` reads slots back, ``recurrent_kda`` takes one decode
  step straight from the pool.

``run`` computes the plain form in 32 bits (64 where a quotient is rounded to
a whole number), or calls the framework where ``own`` is true.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
CONV = 4  # ShortConv taps (three inputs of history)
EPS = 1e-6
TINY = 2.0 ** -100  # a group whose largest magnitude is below this counts as zeros


def listed():
    return [
        # a layer's entry in the training of one long sequence of a wide model
        {"name": "norm_train", "kind": "norm", "quant": False, "dtype": "bf16", "rows": 8192, "width": 7168, "group": 0},
        # the same for a short batch of odd width in full precision: latency
        {"name": "norm_train_odd", "kind": "norm", "quant": False, "dtype": "f32", "rows": 333, "width": 1001, "group": 0},
        # a decode step's entry, 8 bits with one scale a token: latency
        {"name": "norm_quant_decode", "kind": "norm", "quant": True, "dtype": "bf16", "rows": 32, "width": 2048,
         "group": 0},
        # a prefill's entry, 8 bits with one scale per 128 channels
        {"name": "norm_quant_prefill", "kind": "norm", "quant": True, "dtype": "bf16", "rows": 8192, "width": 4096,
         "group": 128},
        # one user's next token through a projection with that user's adapter
        {"name": "adapters_one", "kind": "adapters", "dtype": "bf16", "batch": 1, "tokens": 1, "d_in": 2048,
         "d_out": 2048, "rank": 16, "adapters": 4},
        # a full serving batch's next token, 48 adapters in the batch
        {"name": "adapters_decode", "kind": "adapters", "dtype": "bf16", "batch": 200, "tokens": 1, "d_in": 4096,
         "d_out": 4096, "rank": 32, "adapters": 48},
        # the verification of a draft of five tokens, sizes off every vector and tile
        {"name": "adapters_verify", "kind": "adapters", "dtype": "f16", "batch": 24, "tokens": 5, "d_in": 1001,
         "d_out": 777, "rank": 12, "adapters": 9},
        # prompts of five requests
        {"name": "adapters_prefill", "kind": "adapters", "dtype": "bf16", "batch": 5, "tokens": 1639, "d_in": 2048,
         "d_out": 2048, "rank": 16, "adapters": 8},
        # sequences put to rest: eight layers' caches of 32 sequences into a pool
        {"name": "store_layers", "kind": "store", "layers": 8, "batch": 32, "slots": 48, "heads": 32, "key_dim": 128,
         "value_dim": 128},
        # and brought back
        {"name": "load_layers", "kind": "load", "layers": 8, "batch": 32, "slots": 48, "heads": 32, "key_dim": 128,
         "value_dim": 128},
        # one preempted sequence's next token
        {"name": "resume_one", "kind": "resume", "dtype": "bf16", "batch": 1, "slots": 8, "heads": 16, "key_dim": 128,
         "value_dim": 128},
        # a whole preempted batch's next token
        {"name": "resume_batch", "kind": "resume", "dtype": "bf16", "batch": 256, "slots": 320, "heads": 32,
         "key_dim": 128, "value_dim": 128},
    ]


def _spread(rng, low, high):
    """A whole number spread over the logarithm of low..high."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "adapters", "adapters", "adapters", "store", "load", "resume"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "norm":
        quant = rng.random() < 0.5
        width = rng.choice([_spread(rng, 40, 8192), 64 * _spread(rng, 2, 128)])
        group = rng.choice([0, 0, 32, 64, 128]) if quant else 0
        if group:
            width = max(1, width // group) * group
        return {"kind": "norm", "quant": quant, "dtype": dtype, "group": group, "width": width,
                "rows": _spread(rng, 1, max(2, 8192 * 7168 // (2 * width) if width > 512 else 30000))}
    if kind == "adapters":
        d_in, d_out = (rng.choice([_spread(rng, 100, 4096), 64 * _spread(rng, 2, 64)]) for _ in range(2))
        tokens = rng.choice([1, 1, rng.randint(2, 8), _spread(rng, 16, 1500)])
        batch = _spread(rng, 1, 256) if tokens < 16 else rng.randint(1, 6)
        return {"kind": "adapters", "dtype": dtype, "batch": batch, "tokens": tokens, "d_in": d_in, "d_out": d_out,
                "rank": rng.choice([4, 8, 12, 16, 16, 32, 64]), "adapters": _spread(rng, 1, 64)}
    key_dim, value_dim = rng.choice([(128, 128), (128, 128), (64, 64), (64, 128), (96, 96), (40, 50)])
    heads = rng.choice([4, 6, 8, 16, 32])
    batch = _spread(rng, 1, 256 if kind == "resume" else 32)
    case = {"kind": kind, "batch": batch, "slots": batch + rng.randint(0, batch), "heads": heads, "key_dim": key_dim,
            "value_dim": value_dim}
    return {**case, "dtype": dtype} if kind == "resume" else {**case, "layers": rng.randint(1, 8)}


# ---- inputs -------------------------------------------------------------------


def _normal(gen, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=gen, device="cuda") * std).to(dtype)


def _states(case, gen):
    """The decode caches of the layers, stacked: f32 states whose key channels
    have magnitudes of their own (slow channels hold more than fast ones)."""
    L, B, H, K, V = case["layers"], case["batch"], case["heads"], case["key_dim"], case["value_dim"]
    size = torch.exp(_normal(gen, L, B, H, K, 1)) * 0.02
    return {
        "recurrent": _normal(gen, L, B, H, K, V) * size,
        "q": _normal(gen, L, B, CONV - 1, H * K, dtype=torch.bfloat16),
        "k": _normal(gen, L, B, CONV - 1, H * K, dtype=torch.bfloat16),
        "v": _normal(gen, L, B, CONV - 1, H * V, dtype=torch.bfloat16),
        "offset": torch.randint(1, 8192, (L, B), generator=gen, device="cuda"),
    }


def _pool(case, gen, fill):
    """A pool of slots, stacked over the layers: packed states as an earlier store left them (or empty)."""
    L, N, H, K, V = case.get("layers", 1), case["slots"], case["heads"], case["key_dim"], case["value_dim"]
    if fill:
        values = torch.randint(-127, 128, (L, N, H, K, V), generator=gen, device="cuda", dtype=torch.int8)
        scales = torch.exp(_normal(gen, L, N, H, K)) * 4e-4
    else:
        values = torch.zeros(L, N, H, K, V, device="cuda", dtype=torch.int8)
        scales = torch.zeros(L, N, H, K, device="cuda")
    rest = lambda w: (_normal(gen, L, N, CONV - 1, w, dtype=torch.bfloat16) if fill else  # noqa: E731
                      torch.zeros(L, N, CONV - 1, w, device="cuda", dtype=torch.bfloat16))
    return {"values": values, "scales": scales, "q": rest(H * K), "k": rest(H * K), "v": rest(H * V),
            "offset": torch.randint(1, 8192, (L, N), generator=gen, device="cuda")}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]
    if kind == "norm":
        dt, shape = DTYPES[case["dtype"]], (case["rows"], case["width"])
        s = {"case": case, "x": _normal(gen, *shape, dtype=dt), "residual": _normal(gen, *shape, std=2.0, dtype=dt),
             "weight": (1 + _normal(gen, case["width"], std=0.1)).to(dt)}
        if not case["quant"]:
            s["dy"], s["dh"] = _normal(gen, *shape, dtype=dt), _normal(gen, *shape, dtype=dt)
        return s
    if kind == "adapters":
        dt, n, r = DTYPES[case["dtype"]], case["adapters"], case["rank"]
        d_in, d_out, batch = case["d_in"], case["d_out"], case["batch"]
        ids = torch.randint(0, n, (batch,), generator=gen, device="cuda")
        if batch > 3:  # some requests have no adapter
            ids[torch.randperm(batch, generator=gen, device="cuda")[: batch // 8 + 1]] = -1
        return {"case": case, "ids": ids, "x": _normal(gen, batch, case["tokens"], d_in, dtype=dt),
                "weight": _normal(gen, d_out, d_in, std=d_in ** -0.5, dtype=dt),
                "bias": _normal(gen, d_out, std=0.1, dtype=dt),
                "a": _normal(gen, n, r, d_in, std=d_in ** -0.5, dtype=dt),
                "b": _normal(gen, n, d_out, r, std=0.3 * r ** -0.5, dtype=dt),
                "scaling": 0.5 + torch.rand(n, generator=gen, device="cuda")}
    slots = torch.randperm(case["slots"], generator=gen, device="cuda")[: case["batch"]]
    if kind == "store":
        return {"case": case, "slots": slots, "states": _states(case, gen), "pool": _pool(case, gen, False)}
    if kind == "load":
        return {"case": case, "slots": slots, "pool": _pool(case, gen, True)}
    # one token: q and k L2-normalised, decays from slow to fast, beta a sigmoid
    dt, B, H, K, V = DTYPES[case["dtype"]], case["batch"], case["heads"], case["key_dim"], case["value_dim"]
    q, k = (_normal(gen, B, 1, H, K) for _ in range(2))
    q, k = (t / t.square().sum(-1, keepdim=True).sqrt() for t in (q, k))
    spread = torch.linspace(-5, 0, K, device="cuda")
    g = -5 / (1 + torch.exp(-(spread + _normal(gen, B, 1, H, K, std=0.5))))
    beta = 1 / (1 + torch.exp(-_normal(gen, B, 1, H)))
    return {"case": case, "slots": slots, "pool": _pool(case, gen, True), "q": q.to(dt), "k": k.to(dt),
            "v": _normal(gen, B, 1, H, V, dtype=dt), "g": g.to(dt), "beta": beta.to(dt)}


# ---- the framework's calls ------------------------------------------------------


def _kda():
    root = str(Path(__file__).resolve().parents[1] / "kimi-k3-pytorch_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    import kda

    return kda


def _own_norm(kda, s):
    case = s["case"]
    if case["quant"]:
        q, scales, h = kda.fused.add_rmsnorm_quant(s["x"], s["residual"], s["weight"], EPS,
                                                   group_size=case["group"] or None)
        return {"q": q, "scales": scales, "h": h}
    leaves = [s[n].detach().requires_grad_() for n in ("x", "residual", "weight")]
    y, h = kda.fused.add_rmsnorm(*leaves, EPS)
    dx, dr, dw = torch.autograd.grad((y, h), leaves, (s["dy"], s["dh"]))
    return {"y": y, "h": h, "dx": dx, "dr": dr, "dw": dw}


def _own_packed(kda, pool):
    """The pool's layers as the framework's objects."""
    state, conv = kda.state, kda.ShortConvState
    return [state.PackedKDAState(state.PackedState(values, scales), conv(q), conv(k), conv(v), offset)
            for values, scales, q, k, v, offset in zip(*(pool[n].unbind(0) for n in ("values", "scales", "q", "k", "v",
                                                                                      "offset")))]


def _own(s):
    kda = _kda()
    kind = s["case"]["kind"]
    if kind == "norm":
        return _own_norm(kda, s)
    if kind == "adapters":
        stack = kda.adapters.AdapterStack(s["a"], s["b"], s["scaling"])
        return kda.adapters.adapter_linear(s["x"], s["weight"], s["bias"], stack, s["ids"])
    if kind == "store":
        conv, x = kda.ShortConvState, s["states"]
        states = [kda.KDAState(r, conv(q), conv(k), conv(v), offset) for r, q, k, v, offset in
                  zip(*(x[n].unbind(0) for n in ("recurrent", "q", "k", "v", "offset")))]
        kda.cache.pack_states(states, out=_own_packed(kda, s["pool"]), slots=s["slots"])
        return s["pool"]
    if kind == "load":
        states = kda.cache.unpack_states(_own_packed(kda, s["pool"]), slots=s["slots"])
        return [{"recurrent": t.recurrent_state, "q": t.q_conv_state.buffer, "k": t.k_conv_state.buffer,
                 "v": t.v_conv_state.buffer, "offset": t.sequence_offset} for t in states]
    packed = kda.state.PackedState(s["pool"]["values"][0], s["pool"]["scales"][0])
    out = kda.recurrent_kda(s["q"], s["k"], s["v"], s["g"], s["beta"], packed, True, state_slots=s["slots"])
    return {"o": out.hidden_states, "state": out.final_state}


# ---- the plain forms --------------------------------------------------------------


def _groups(y, group):
    return y.reshape(y.shape[0], -1, group or y.shape[1])


def _plain_norm(s):
    case, dt = s["case"], DTYPES[s["case"]["dtype"]]
    h = (s["x"].float() + s["residual"].float()).to(dt)
    hf, w = h.float(), s["weight"].float()
    inv = torch.rsqrt(hf.square().mean(-1, keepdim=True) + EPS)
    y = hf * inv * w
    if case["quant"]:
        y = _groups(y, case["group"])
        amax = y.abs().amax(-1, keepdim=True)
        zero = amax < TINY
        scales = torch.where(zero, torch.zeros_like(amax), amax / 448)
        q = torch.where(zero, torch.zeros_like(y), y / torch.where(zero, torch.ones_like(amax), scales))
        return {"q": q.reshape(h.shape).to(torch.float8_e4m3fn), "scales": scales[..., 0], "h": h}
    dy, dh = s["dy"].float(), s["dh"].float()
    wdy = dy * w
    dx = dh + inv * (wdy - hf * inv.square() * (wdy * hf).mean(-1, keepdim=True))
    dx = dx.to(dt)
    return {"y": y.to(dt), "h": h, "dx": dx, "dr": dx, "dw": (dy * hf * inv).sum(0).to(dt)}


def _plain_adapters(s):
    case = s["case"]
    n, r = case["adapters"], case["rank"]
    x = s["x"].float().reshape(-1, case["d_in"])
    ids = s["ids"].repeat_interleave(case["tokens"])
    # every adapter's product, and of them each row's own
    pick = (ids[:, None] == torch.arange(n, device=ids.device)).float() * s["scaling"]
    low = (x @ s["a"].float().reshape(n * r, -1).t()).reshape(-1, n, r) * pick[..., None]
    wide = s["b"].float().transpose(1, 2).reshape(n * r, -1)
    y = x @ s["weight"].float().t() + s["bias"].float() + low.reshape(-1, n * r) @ wide
    return y.to(s["x"].dtype).reshape(*s["x"].shape[:-1], -1)


def _plain_store(s):
    x, pool, slots = s["states"], s["pool"], s["slots"]
    amax = x["recurrent"].abs().amax(-1)
    zero = amax < TINY
    scales = torch.where(zero, torch.zeros_like(amax), amax / 127)
    whole = torch.where(zero, torch.ones_like(amax), scales).double()[..., None]
    values = torch.round(x["recurrent"].double() / whole).clamp(-127, 127)  # ties to even
    values = torch.where(zero[..., None], torch.zeros_like(values), values)
    pool["values"][:, slots] = values.to(torch.int8)
    pool["scales"][:, slots] = scales
    for n in ("q", "k", "v", "offset"):
        pool[n][:, slots] = x[n]
    return pool


def _plain_load(s):
    pool, slots = s["pool"], s["slots"]
    got = {n: pool[n][:, slots].unbind(0) for n in ("q", "k", "v", "offset")}
    got["recurrent"] = (pool["values"][:, slots].float() * pool["scales"][:, slots][..., None]).unbind(0)
    return [dict(zip(got, layer)) for layer in zip(*got.values())]


def _step(s, dt):
    """One token of the recurrence from the pool's states, in `dt`."""
    slots = s["slots"]
    state = s["pool"]["values"][0][slots].to(dt) * s["pool"]["scales"][0][slots].to(dt)[..., None]
    q, k, v, g, beta = (s[n][:, 0].to(dt) for n in ("q", "k", "v", "g", "beta"))
    state = state * torch.exp(g)[..., None]
    error = v - (state * k[..., None]).sum(-2)
    state = state + (beta[..., None] * k)[..., None] * error[..., None, :]
    return {"o": (state * q[..., None]).sum(-2)[:, None], "state": state}


def _plain_resume(s):
    out = _step(s, torch.float32)
    return {"o": out["o"].to(s["v"].dtype), "state": out["state"]}


def run(state):
    if own:
        return _own(state)
    return {"norm": _plain_norm, "adapters": _plain_adapters, "store": _plain_store, "load": _plain_load,
            "resume": _plain_resume}[state["case"]["kind"]](state)


# ---- what a pass cannot do without ------------------------------------------------


def work(case):
    kind = case["kind"]
    if kind == "norm":
        n, e = case["rows"] * case["width"], DTYPES[case["dtype"]].itemsize
        if case["quant"]:  # x, residual; h, q, the scales
            scales = 4 * (n // case["group"] if case["group"] else case["rows"])
            return {"bytes": 3 * n * e + n + scales + case["width"] * e, "flops": 8 * n}
        return {"bytes": 7 * n * e + 2 * case["width"] * e, "flops": 20 * n}  # x, residual, dy, dh; y, h, dx
    if kind == "adapters":
        e, rows, used = DTYPES[case["dtype"]].itemsize, case["batch"] * case["tokens"], min(case["adapters"],
                                                                                             case["batch"])
        d_in, d_out, r = case["d_in"], case["d_out"], case["rank"]
        return {"bytes": e * (rows * (d_in + d_out) + d_in * d_out + used * r * (d_in + d_out)),
                "flops": 2 * rows * (d_in * d_out + r * (d_in + d_out))}
    H, K, V, B = case["heads"], case["key_dim"], case["value_dim"], case["batch"]
    n = B * H * K * V
    if kind == "resume":
        e = DTYPES[case["dtype"]].itemsize
        return {"bytes": 5 * n + 4 * B * H * K + e * B * H * (3 * K + 2 * V + 1), "flops": 9 * n}
    conv = 2 * B * (CONV - 1) * H * (2 * K + V)
    return {"bytes": case["layers"] * (5 * n + 4 * B * H * K + 2 * (conv + 8 * B)), "flops": 2 * case["layers"] * n}


# ---- the definitions in 64 bits -----------------------------------------------------


def _exact_norm(s):
    case, dt = s["case"], DTYPES[s["case"]["dtype"]]
    total = s["x"].double() + s["residual"].double()
    h, w = total.to(dt).double(), s["weight"].double()  # the norm reads the stored sum
    norm = 1 / torch.sqrt((h * h).sum(1) / h.shape[1] + EPS)
    y = torch.einsum("rc,r,c->rc", h, norm, w)
    if case["quant"]:
        blocks = y.unflatten(1, (-1, case["group"] or h.shape[1]))
        scales = blocks.abs().max(2).values / 448
        return {"q": (blocks / scales[:, :, None]).flatten(1), "scales": scales, "h": total}
    dy = s["dy"].double()
    # d/dh of sum(dy y): the norm's own factor, and what the row's mean square gives back
    back = torch.einsum("rc,c,r->rc", dy, w, norm)
    mean = torch.einsum("rc,rc->r", back, h) / h.shape[1]
    dx = s["dh"].double() + back - h * (norm ** 2 * mean)[:, None]
    return {"y": y, "h": total, "dx": dx, "dr": dx, "dw": torch.einsum("rc,rc,r->c", dy, h, norm)}


def _exact_adapters(s):
    x = s["x"].double()
    y = torch.matmul(x, s["weight"].double().t()) + s["bias"].double()
    for i, adapter in enumerate(s["ids"].tolist()):
        if adapter >= 0:
            low = torch.matmul(x[i], s["a"][adapter].double().t())
            y[i] += s["scaling"][adapter].double() * torch.matmul(low, s["b"][adapter].double().t())
    return y


def _exact_store(s):
    x, slots, pool = s["states"], s["slots"].tolist(), s["pool"]
    scales = pool["scales"].double()
    got = {n: pool[n].clone() for n in ("q", "k", "v")}
    for row, slot in enumerate(slots):
        scales[:, slot] = x["recurrent"][:, row].double().abs().max(-1).values / 127
        for n in got:
            got[n][:, slot] = x[n][:, row]
    return {"values": None, "scales": scales, "offset": None, **got}


def _exact_load(s):
    pool, slots = s["pool"], s["slots"].tolist()
    layers = []
    for i in range(s["case"]["layers"]):
        rows = [pool["values"][i, j].double() * pool["scales"][i, j].double().unsqueeze(-1) for j in slots]
        layers.append({"recurrent": torch.stack(rows), "offset": None,
                       **{n: torch.stack([pool[n][i, j] for j in slots]).double() for n in ("q", "k", "v")}})
    return layers


def _exact_resume(s):
    slots = s["slots"].tolist()
    outputs, states = [], []
    for row, slot in enumerate(slots):
        old = s["pool"]["values"][0, slot].double() * s["pool"]["scales"][0, slot].double().unsqueeze(-1)  # [H,K,V]
        q, k, v, g, beta = (s[n][row, 0].double() for n in ("q", "k", "v", "g", "beta"))
        kept = old * g.exp().unsqueeze(-1)
        recall = torch.einsum("hkv,hk->hv", kept, k)
        new = kept + torch.einsum("h,hk,hv->hkv", beta, k, v - recall)
        outputs.append(torch.einsum("hkv,hk->hv", new, q))
        states.append(new)
    return {"o": torch.stack(outputs).unsqueeze(1), "state": torch.stack(states)}


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "adapters": _exact_adapters, "store": _exact_store, "load": _exact_load,
            "resume": _exact_resume}[case["kind"]](s)
