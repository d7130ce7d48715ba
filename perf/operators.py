"""Cases of the attention whose state decays head by head, and of the states that it leaves behind.

With q, k (Dk), v, y (Dv) and the log decay g of one head, and S (Dk, Dv) that head's state:

    S_t = exp(g_t) S_{t-1} + k_t v_t^T          y_t = scale * S_t^T q_t

Kinds
  prompt   y and the last states of whole sequences (rows of a batch, or packed behind each other)
  train    the same, and the gradients of q, k, v, g and of the first states
  step     one more token for each of N sequences, whose states are pages of a pool that is updated in place
  pages    pages of such a pool copied, forked, moved together and cleared by one list of (from, to)

`run` computes them in elementary torch operations, or with `own` through the package's entry points.
"""
import math

import numpy as np
import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
_DEV = "cuda"
_L = 64                                                  # tokens of a chunk of the plain form


def listed():
    return [
        # one image's tokens through a small layer with a fixed decay for each head: the smallest prompt, all latency
        dict(name="prompt_one_image", kind="prompt", N=1, T=196, H=3, Hq=3, Hk=3, Hv=3, Dk=64, Dv=64, dtype="bf16", g="head", packed=False, state=False),
        # a batch of images through a base-size layer, decays from the data
        dict(name="prompt_base", kind="prompt", N=64, T=196, H=12, Hq=12, Hk=12, Hv=12, Dk=64, Dv=64, dtype="bf16", g="fp32", packed=False, state=False),
        # a server's batch of prompts of all lengths, packed, that go on from earlier states; queries and keys shared by four heads each
        dict(name="prompts_packed_shared", kind="prompt", N=48, T=2048, H=16, Hq=4, Hk=4, Hv=16, Dk=128, Dv=64, dtype="bf16", g="fp32", packed=True, state=True),
        # dense prediction: two images of about 1333 x 800 in fp32
        dict(name="prompt_dense_fp32", kind="prompt", N=2, T=4150, H=12, Hq=12, Hk=12, Hv=12, Dk=64, Dv=64, dtype="fp32", g="fp32", packed=False, state=False),
        # a few very long sequences
        dict(name="prompt_long_fp16", kind="prompt", N=4, T=16384, H=12, Hq=12, Hk=12, Hv=12, Dk=64, Dv=64, dtype="fp16", g="fp32", packed=False, state=True),
        # one layer's operator in bf16 training of a base-size model
        dict(name="train_base", kind="train", N=64, T=196, H=12, Hq=12, Hk=12, Hv=12, Dk=64, Dv=64, dtype="bf16", g="fp32", packed=False, state=False),
        # detection fine-tuning: two large images, fp32
        dict(name="train_dense_fp32", kind="train", N=2, T=4150, H=12, Hq=12, Hk=12, Hv=12, Dk=64, Dv=64, dtype="fp32", g="fp32", packed=False, state=False),
        # fine-tuning at 384 x 384 with a class token: head sizes that fill no tile, shared keys, one decay a head, first states that learn
        dict(name="train_odd_heads", kind="train", N=8, T=577, H=6, Hq=6, Hk=2, Hv=6, Dk=48, Dv=80, dtype="fp16", g="head", packed=False, state=True),
        # the next token of one sequence: latency
        dict(name="step_one", kind="step", N=1, P=4, H=12, Hq=12, Hk=12, Hv=12, Dk=64, Dv=64, dtype="bf16", g="fp32"),
        # the next token of a server's whole batch
        dict(name="step_batch", kind="step", N=512, P=640, H=12, Hq=12, Hk=12, Hv=12, Dk=64, Dv=64, dtype="bf16", g="fp32"),
        # one prompt's state forked to the beams that go on from it
        dict(name="pages_fork", kind="pages", M=16, P=64, H=12, Dk=64, Dv=64, how="fork"),
        # a pool moved together after sequences ended: every page that stays moves down, over pages that move as well
        dict(name="pages_compact", kind="pages", M=700, P=1024, H=12, Dk=64, Dv=64, how="compact"),
    ]


def _log_int(rng, lo, hi):
    """A whole number spread evenly over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["prompt", "prompt", "train", "train", "step", "pages"])
    H = rng.choice([3, 6, 12, 16]) if rng.random() < 0.7 else rng.randint(1, 20)
    size = lambda: 64 if rng.random() < 0.5 else rng.choice([32, 128]) if rng.random() < 0.5 else rng.randint(8, 128)  # noqa: E731
    Dk, Dv = size(), size()
    if kind == "pages":
        how = rng.choice(["fork", "compact", "permute", "clear"])
        P = _log_int(rng, 8, max(8, min(1024, 1024 * 12 * 4096 // (H * Dk * Dv))))
        M = rng.randint(1, P // 2) if how in ("fork", "clear") else rng.randint(2, P * 3 // 4)
        return dict(kind=kind, M=M, P=P, H=H, Dk=Dk, Dv=Dv, how=how)
    shared = lambda: H if rng.random() < 0.7 else rng.choice([d for d in range(1, H + 1) if H % d == 0])  # noqa: E731
    heads = dict(H=H, Hq=shared(), Hk=shared(), Hv=shared(), Dk=Dk, Dv=Dv)
    dtype = rng.choice(["bf16", "fp16", "fp32"])
    if kind == "step":
        N = _log_int(rng, 1, max(1, min(512, 512 * 12 * 4096 // (H * Dk * Dv))))
        return dict(kind=kind, N=N, P=N + rng.randint(0, N // 2 + 3), **heads, dtype=dtype, g=rng.choice(["fp32", "head", dtype]))
    # one token up to long sequences; the cost goes by tokens, heads and the larger of the head sizes' tiles
    most = (2 * 4150 * 12 if kind == "train" else 4 * 16384 * 12) // (H * (2 if max(Dk, Dv) > 64 else 1)) // (2 if dtype == "fp32" and kind == "prompt" else 1)
    T = _log_int(rng, 1, min(16384 if kind == "prompt" else 4150, most))
    N = _log_int(rng, 1, max(1, min(64, most // T)))
    return dict(kind=kind, N=N, T=T, **heads, dtype=dtype, g=rng.choice(["fp32", "fp32", "head", dtype]), packed=rng.random() < 0.4, state=rng.random() < 0.5)


# ---- inputs ----------------------------------------------------------------------------------------------------------

def _lengths(case):
    """The lengths of a packed case's sequences, the same for every seed: spread over the logarithm of 1 .. T, one of them T, and one empty where
    there are several."""
    r = np.random.default_rng(case["N"] * 100_000 + case["T"])
    n = np.maximum(1, np.round(case["T"] ** r.random(case["N"]))).astype(np.int64)
    n[r.integers(case["N"])] = case["T"]
    if case["N"] > 2:
        n[(int(np.argmax(n)) + 1) % case["N"]] = 0
    return n


def _inputs(case, seed):
    gen = torch.Generator(_DEV).manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=gen, device=_DEV)  # noqa: E731
    dt = _DTYPES[case["dtype"]]
    H, Dk, Dv = case["H"], case["Dk"], case["Dv"]
    rows = (case["N"],)
    s = {"case": case, "scale": Dk ** -0.5}
    if case["kind"] != "step":
        rows = (case["N"], case["T"])
        if case["packed"]:
            n = _lengths(case)
            rows = (1, int(n.sum()))
            s["offsets"] = torch.from_numpy(np.concatenate([[0], np.cumsum(n)])).to(device=_DEV, dtype=torch.int32)
            s["longest"] = int(n.max())
    s["q"] = normal(*rows, case["Hq"], Dk).to(dt)
    s["k"] = normal(*rows, case["Hk"], Dk).to(dt)
    s["v"] = normal(*rows, case["Hv"], Dv).to(dt)
    # heads that forget within a few tokens up to heads that keep a thousand
    base = torch.linspace(math.log(0.3), math.log(1e-3), H, device=_DEV)
    if case["g"] == "head":
        s["g"] = -torch.exp(base + 0.1 * normal(H))
    else:
        s["g"] = (-torch.exp(base + 0.8 * normal(*rows, H))).to(_DTYPES[case["g"]])
    return s, normal


def _page_list(case, seed):
    r = np.random.default_rng(seed)
    P, M, how = case["P"], case["M"], case["how"]
    if how == "fork":                                    # one page to M others
        p = r.permutation(P)
        return np.full(M, p[0]), p[1:M + 1]
    if how == "clear":                                   # freed pages, cleared for the next sequences
        return np.full(M, -1), r.permutation(P)[:M]
    if how == "permute":
        p = r.permutation(P)[:M]
        return p, np.roll(p, 1)
    keep = np.sort(r.permutation(P)[:M])                 # the pages that stay, in order, to the front
    return keep, np.arange(M)


def prepare(case, seed):
    if case["kind"] == "pages":
        gen = torch.Generator(_DEV).manual_seed(seed)
        src, dst = _page_list(case, seed)
        return {"case": case, "pool": torch.randn(case["P"], case["H"], case["Dk"], case["Dv"], generator=gen, device=_DEV),
                "src": torch.from_numpy(src.astype(np.int32)).to(_DEV), "dst": torch.from_numpy(dst.astype(np.int32)).to(_DEV)}
    s, normal = _inputs(case, seed)
    H, Dk, Dv = case["H"], case["Dk"], case["Dv"]
    if case["kind"] == "step":
        s["pool"] = normal(case["P"], H, Dk, Dv)
        s["slots"] = torch.from_numpy(np.random.default_rng(seed).permutation(case["P"])[:case["N"]].astype(np.int32)).to(_DEV)
        return s
    s["state"] = normal(case["N"], H, Dk, Dv) if case["state"] else None
    if case["kind"] == "train":
        s["gy"] = normal(*s["q"].shape[:2], H, Dv).to(s["q"].dtype)
        s["gstate"] = normal(case["N"], H, Dk, Dv) if case["state"] else None
        s["leaves"] = [s[n].requires_grad_() for n in ("q", "k", "v", "g", "state") if s[n] is not None]
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------

def run(s):
    case = s["case"]
    if case["kind"] == "pages":
        return _own_pages(s) if own else _plain_pages(s)
    if case["kind"] == "step":
        return _own_step(s) if own else _plain_step(s)
    if case["kind"] == "prompt":
        return _own_prompt(s) if own else _plain_prompt(s)
    y, last = _own_prompt(s) if own else _plain_prompt(s)
    if s["gstate"] is None:
        grads = torch.autograd.grad(y, s["leaves"], s["gy"])
    else:
        grads = torch.autograd.grad((y, last), s["leaves"], (s["gy"], s["gstate"]))
    return [y.detach(), last.detach(), *grads]


def _own_prompt(s):
    import vision_rwkv_amd as vr
    return vr.decay_attention(s["q"], s["k"], s["v"], s["g"], scale=s["scale"], state=s["state"], offsets=s.get("offsets"), return_state=True)


def _own_step(s):
    import vision_rwkv_amd as vr
    return vr.decay_attention_step(s["q"], s["k"], s["v"], s["g"], s["pool"], s["slots"], scale=s["scale"]), s["pool"]


def _own_pages(s):
    import vision_rwkv_amd as vr
    return vr.copy_states(s["pool"], s["src"], s["dst"])


def _heads(x, H):
    """x (..., h, D) in fp32 with each of its h heads repeated for the H / h that share it."""
    return x.float().repeat_interleave(H // x.shape[-2], -2)


def _plain_prompt(s):
    case = s["case"]
    H = case["H"]
    q, k, v = (_heads(s[n], H) for n in ("q", "k", "v"))
    g = s["g"].double()
    g = g.expand(*q.shape[:2], H) if case["g"] == "head" else g
    if not case["packed"]:
        y, last = _chunked(q, k, v, g, s["scale"], s["state"])
        return y.to(s["q"].dtype), last
    # packed sequences as rows of a padded batch, and back
    off = s["offsets"].long()
    length = off[1:] - off[:-1]
    t = torch.arange(s["longest"], device=off.device)
    inside = t < length[:, None]
    at = torch.where(inside, off[:-1, None] + t, 0)
    pad = lambda x: torch.where(inside.reshape(*inside.shape, *(1,) * (x.dim() - 2)), x[0][at], 0)  # noqa: E731
    y, last = _chunked(pad(q), pad(k), pad(v), pad(g), s["scale"], s["state"])
    row = torch.arange(q.shape[1], device=off.device)
    n = torch.searchsorted(off[1:], row, right=True)
    return y[n, row - off[n]][None].to(s["q"].dtype), last


def _chunked(q, k, v, g, scale, state):
    """Rows (N, T, H, .) in chunks of _L tokens: the products of a chunk's tokens with each other under their decays, and its first state, which is
    the sum over all chunks before it."""
    N, T, H, Dk = q.shape
    Dv, C = v.shape[-1], -(-T // _L)
    cut = lambda x: torch.nn.functional.pad(x, (0, 0) * (x.dim() - 2) + (0, C * _L - T)).reshape(N, C, _L, *x.shape[2:]).movedim(3, 2)  # noqa: E731
    q, k, v, G = cut(q), cut(k), cut(v), cut(g).cumsum(-1)                                # (N, C, H, L, .)
    ahead = torch.ones(_L, _L, dtype=torch.bool, device=q.device).tril()
    decay = torch.exp((G[..., :, None] - G[..., None, :]).masked_fill(~ahead, -math.inf)).float()
    inner = (scale * (q @ k.transpose(-1, -2)) * decay) @ v
    own_part = (k * torch.exp(G[..., -1:] - G).float()[..., None]).transpose(-1, -2) @ v   # (N, C, H, Dk, Dv)
    total = torch.cat([torch.zeros_like(G[:, :1, :, -1]), G[..., -1].cumsum(1)], 1)        # (N, C + 1, H): decay in front of each chunk
    far = (total[:, :, None] - total[:, None, 1:]).permute(0, 3, 1, 2)                     # (N, H, C + 1, C)
    before = torch.ones(C + 1, C, dtype=torch.bool, device=q.device).tril(-1)
    far = torch.exp(far.masked_fill(~before, -math.inf)).float()
    S = (far @ own_part.movedim(2, 1).reshape(N, H, C, Dk * Dv)).reshape(N, H, C + 1, Dk, Dv)
    if state is not None:
        S = S + torch.exp(total).float().movedim(2, 1)[..., None, None] * state[:, :, None]
    outer = scale * torch.exp(G).float()[..., None] * (q @ S[:, :, :C].movedim(1, 2))
    y = (inner + outer).movedim(2, 3).reshape(N, C * _L, H, Dv)[:, :T]
    return y, S[:, :, C].contiguous()


def _plain_step(s):
    H, slots = s["case"]["H"], s["slots"].long()
    q, k, v = (_heads(s[n], H) for n in ("q", "k", "v"))
    S = torch.exp(s["g"].float())[..., None, None] * s["pool"][slots] + k[..., :, None] * v[..., None, :]
    s["pool"][slots] = S
    return (s["scale"] * (q[..., :, None] * S).sum(-2)).to(s["q"].dtype), s["pool"]


def _plain_pages(s):
    src, dst = s["src"].long(), s["dst"].long()
    some = (src >= 0)[:, None, None, None]
    s["pool"][dst] = torch.where(some, s["pool"][src.clamp(min=0)], 0)
    return s["pool"]


# ---- what a pass cannot do without -----------------------------------------------------------------------------------

def work(case):
    if case["kind"] == "pages":
        page = case["H"] * case["Dk"] * case["Dv"] * 4
        read = {"fork": 1, "clear": 0}.get(case["how"], case["M"])
        return {"bytes": page * (read + case["M"]), "flops": 0}
    H, Dk, Dv, e = case["H"], case["Dk"], case["Dv"], _BYTES[case["dtype"]]
    if case["kind"] == "step":
        rows, states = case["N"], 2 * case["N"]
    else:
        rows = case["N"] * case["T"] if not case["packed"] else int(_lengths(case).sum())
        states = case["N"] * (2 if case["state"] else 1)
    gate = H * 4 if case["g"] == "head" else rows * H * _BYTES[case["g"]]
    q, k, v, y = (rows * n * e for n in (case["Hq"] * Dk, case["Hk"] * Dk, case["Hv"] * Dv, H * Dv))
    moved = q + k + v + y + gate + states * H * Dk * Dv * 4
    if case["kind"] == "train":                          # gy read, four gradients (and the first states') written
        moved += y + q + k + v + gate + (2 * case["N"] * H * Dk * Dv * 4 if case["state"] else 0)
    # a product of a state and a vector, or of two vectors to a state, for each token and head: 2 forward; S again, its gradient, dq, dk, dv backward
    return {"bytes": moved, "flops": rows * H * 2 * Dk * Dv * (7 if case["kind"] == "train" else 2)}


# ---- the definition, token by token, in 64 bits ----------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "pages":
        pool = s["pool"].double().cpu().numpy()
        out = pool.copy()
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            out[b] = pool[a] if a >= 0 else 0.0
        return torch.from_numpy(out)
    with torch.no_grad():
        return _exact_step(s) if case["kind"] == "step" else _exact_rows(s)


def _wide(x, H):
    """x (..., h, D) in 64 bits, head i being head i // (H / h) of x."""
    which = torch.arange(H, device=x.device) // (H // x.shape[-2])
    return x.detach().double().index_select(-2, which)


def _exact_step(s):
    H, pool, y = s["case"]["H"], s["pool"].double(), []
    q, k, v = _wide(s["q"], H), _wide(s["k"], H), _wide(s["v"], H)
    g = s["g"].double().expand(q.shape[0], H)
    for n, slot in enumerate(s["slots"].tolist()):
        pool[slot] = g[n].exp().reshape(H, 1, 1) * pool[slot] + torch.einsum("hk,hv->hkv", k[n], v[n])
        y.append(s["scale"] * torch.einsum("hk,hkv->hv", q[n], pool[slot]))
    return torch.stack(y), pool


def _exact_rows(s):
    """Along the tokens for y and dq = scale S gy, back along them for the state's gradient R, dk = R v and dv = R^T k.  A decay's gradient is what
    crosses it: the sum of q . dq - k . dk over it and the tokens behind it, and what the last state has."""
    case, train = s["case"], s["case"]["kind"] == "train"
    H, scale = case["H"], s["scale"]
    q, k, v = _wide(s["q"], H), _wide(s["k"], H), _wide(s["v"], H)
    rows = q.shape[:2]
    g = s["g"].detach().double().expand(*rows, H)
    y = torch.zeros(*rows, H, case["Dv"], dtype=torch.float64, device=_DEV)
    if case["packed"]:
        off = s["offsets"].tolist()
        first, length = np.array(off[:-1]), np.diff(off)
    else:
        first, length = np.zeros(case["N"], np.int64), np.full(case["N"], case["T"])
    order = np.argsort(-length, kind="stable")           # longest first: the sequences that still have a token t are the first few
    first, length = first[order], length[order]
    row = np.zeros_like(first) if case["packed"] else order
    perm = torch.from_numpy(order).to(_DEV)
    index = [(torch.from_numpy(row).to(_DEV), torch.from_numpy(first).to(_DEV))]
    alive = [int((length > t).sum()) for t in range(int(length.max()))]

    def at(t):
        n = alive[t]
        return n, (index[0][0][:n], index[0][1][:n] + t)

    S = torch.zeros(case["N"], H, case["Dk"], case["Dv"], dtype=torch.float64, device=_DEV)
    if s["state"] is not None:
        S += s["state"].detach().double()[perm]
    if train:
        gy = s["gy"].double()
        dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for t in range(len(alive)):
        n, i = at(t)
        S[:n] = g[i].exp()[..., None, None] * S[:n] + k[i][..., :, None] * v[i][..., None, :]
        y[i] = scale * (q[i][..., None, :] @ S[:n])[..., 0, :]
        if train:
            dq[i] = scale * (S[:n] @ gy[i][..., None])[..., 0]
    last = torch.empty_like(S)
    last[perm] = S
    if not train:
        return y, last
    R = torch.zeros_like(S) if s["gstate"] is None else s["gstate"].double()[perm]
    ends = (R * S).sum((-1, -2))                         # what the last state's gradient brings across every decay of its sequence
    crossing = torch.zeros(case["N"], H, dtype=torch.float64, device=_DEV) + ends
    dg = torch.zeros_like(g)
    for t in reversed(range(len(alive))):
        n, i = at(t)
        R[:n] += scale * q[i][..., :, None] * gy[i][..., None, :]
        dk[i] = (R[:n] @ v[i][..., None])[..., 0]
        dv[i] = (k[i][..., None, :] @ R[:n])[..., 0, :]
        crossing[:n] += (q[i] * dq[i]).sum(-1) - (k[i] * dk[i]).sum(-1)
        dg[i] = crossing[:n]
        R[:n] = g[i].exp()[..., None, None] * R[:n]
    share = lambda d, h: d.reshape(*rows, h, H // h, d.shape[-1]).sum(-2)  # noqa: E731
    dR = torch.empty_like(R)
    dR[perm] = R
    out = [y, last, share(dq, case["Hq"]), share(dk, case["Hk"]), share(dv, case["Hv"]), dg.sum((0, 1)) if case["g"] == "head" else dg]
    return out + ([dR] if s["state"] is not None else [])
