"""Workloads of the operators that serve a MoDA model token by token, and of the rotary positions that its
training and its serving share.

  op "rotary"   rotary positions of a layer's queries and keys: the forward alone, or with its gradients
  op "append"   a prompt's (or one token's) keys and values into a paged cache, the keys rotated on the way
  op "decode"   attention of one new token over its sequence in a paged cache and the L rows of earlier layers
  op "step"     the same with the new token's own key and value: rotated, written to the cache, attended to

  B, T, H, G, D   batch, tokens of a call, KV heads, query heads of a KV head, head dim
  L               depth rows of the new token: one of each earlier layer
  lo, hi          lengths of the sequences: B whole numbers from lo to hi, evenly spread, in a random order
  page, heads     positions of a page; whether a page holds its heads one after another
  rot, pairs      rotated elements of a head; "half" (i, i + rot / 2) or "interleaved" (2 i, 2 i + 1)
  stretch         by how much the positions are stretched for long contexts (frequencies blended between the
                  original and the stretched ones, and a factor on the rotated vectors); 1: not at all
  far             positions are given as a tensor, up to 16 times the sequence's length
"""
import math

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16}


def _case(op, dtype, B, T, H, G, D, **more):
    base = dict(op=op, dtype=dtype, B=B, T=T, H=H, G=G, D=D, L=0, lo=0, hi=0, page=64, heads=True, rot=D, pairs="half",
                stretch=1.0, far=False, train=False)
    return dict(base, **more)


def listed():
    return [
        # positions of one new token each of a small serving batch: what it costs to call the operator at all
        _case("rotary", "bfloat16", 32, 1, 8, 4, 128, far=True, name="rotary_tokens"),
        # the layer's queries and keys of one long prompt
        _case("rotary", "bfloat16", 1, 65536, 8, 4, 128, name="rotary_prompt"),
        # training step of a grouped-query language model
        _case("rotary", "bfloat16", 2, 4096, 4, 4, 128, train=True, name="rotary_train"),
        # training on packed documents in fp16, half of each head rotated, stretched positions, odd length and head count
        _case("rotary", "float16", 3, 1531, 5, 2, 128, rot=64, pairs="interleaved", stretch=4.0, far=True, train=True,
              name="rotary_train_partial"),
        # one new token each of a large serving batch
        _case("append", "bfloat16", 256, 1, 8, 1, 128, lo=1, hi=2048, name="append_tokens"),
        # prompts of different lengths in one padded batch, behind prefixes of different lengths
        _case("append", "bfloat16", 8, 4093, 8, 1, 128, lo=0, hi=512, pairs="interleaved", stretch=4.0, name="append_prompts"),
        # one user, a short context: latency
        _case("decode", "bfloat16", 1, 1, 4, 1, 64, L=4, lo=256, hi=256, page=16, name="decode_one_short"),
        # a serving batch of a grouped-query language model, contexts of all lengths
        _case("decode", "bfloat16", 64, 1, 8, 4, 128, L=32, lo=1, hi=8192, name="decode_batch"),
        # one user, a long context
        _case("decode", "bfloat16", 1, 1, 8, 4, 128, L=32, lo=65536, hi=65536, name="decode_long"),
        # odd sizes: pages that end inside any tile, token-major pages, an empty sequence, narrow heads
        _case("decode", "float16", 37, 1, 5, 2, 64, L=7, lo=0, hi=1531, page=24, heads=False, name="decode_ragged"),
        # a whole decoding step of a layer for one user
        _case("step", "float16", 1, 1, 8, 4, 128, L=32, lo=4095, hi=4095, rot=64, pairs="interleaved", name="step_one"),
        # and for a serving batch
        _case("step", "bfloat16", 64, 1, 4, 4, 128, L=24, lo=1024, hi=4096, stretch=4.0, name="step_batch"),
    ]


MOST_BYTES = 1.3e9      # the largest listed case


def _spread(rng, lo, hi):
    """A whole number from lo to hi, spread over the logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    while True:
        op = rng.choice(["rotary", "append", "decode", "decode", "step"])
        D = rng.choice([64, 128])
        more = dict(rot=rng.choice([r for r in (16, 32, 48, 64, 96, 128, D, D) if r <= D]), pairs=rng.choice(["half", "interleaved"]),
                    stretch=rng.choice([1.0, 1.0, 4.0, 8.0]), page=rng.choice([8, 16, 16, 24, 64, 64, 128, 256]), heads=rng.random() < 0.7)
        if op == "rotary":
            T = _spread(rng, 1, 65536)
            more.update(far=rng.random() < 0.4, train=rng.random() < 0.5)
        elif op == "append":
            T = _spread(rng, 1, 16384)
            more.update(lo=0, hi=_spread(rng, 1, 4096))
        else:
            T = 1
            hi = _spread(rng, 1, 65536)
            more.update(lo=rng.choice([0, 1, hi // 2, hi]), hi=hi, L=rng.choice([0, 1, 4, 7, 11, 24, 32, 64]))
        G = rng.choice([1, 2, 4, 8]) if op != "append" else 1
        case = _case(op, rng.choice(["bfloat16", "bfloat16", "float16"]), _spread(rng, 1, 256), T, rng.randint(1, 16), G, D, **more)
        if work(case)["bytes"] <= MOST_BYTES and case["B"] * (case["hi"] + T) * case["H"] * D <= 2 ** 28:
            return case


def _frequencies(case, device="cpu"):
    """Radians a position for each pair, in 64 bits, and the factor on the rotated vectors.

    Stretched by s (interpolation of the slow pairs, none of the fast ones): a pair that turns more than 32
    times over the original 8192 positions keeps its frequency f, one that turns less than once gets f / s, with a
    linear ramp over the pairs between; vectors grow by 0.1 ln(s) + 1."""
    rot, s = case["rot"], case["stretch"]
    i = torch.arange(rot // 2, dtype=torch.float64, device=device)
    f = 10000.0 ** (-2.0 * i / rot)
    if s == 1.0:
        return f, 1.0
    at = [rot * math.log(8192 / (turns * 2 * math.pi)) / (2 * math.log(10000.0)) for turns in (32.0, 1.0)]
    low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rot - 1)
    ramp = ((i - low) / max(high - low, 1e-3)).clamp(0, 1)
    return f / s * ramp + f * (1 - ramp), 0.1 * math.log(s) + 1.0


def _lengths(case, gen):
    even = torch.linspace(case["lo"], case["hi"], case["B"], dtype=torch.float64).floor().to(torch.int32).cuda()
    return even[torch.randperm(case["B"], generator=gen, device="cuda")]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    B, T, H, G, D, L = (case[x] for x in "BTHGDL")

    def mk(*shape, leaf=False):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype).requires_grad_(leaf)

    inv_freq, factor = _frequencies(case, "cuda")
    s = {"case": case, "inv_freq": inv_freq, "factor": factor}
    if case["op"] == "rotary":
        s["q"], s["k"] = mk(B, T * G, H, D, leaf=case["train"]), mk(B, T, H, D, leaf=case["train"])
        if case["far"]:
            start = torch.randint(0, 16 * max(T, 4096), (B, 1), generator=gen, device="cuda")
            s["positions"] = start + torch.arange(T, device="cuda")
        if case["train"]:
            s["dq"], s["dk"] = mk(B, T * G, H, D), mk(B, T, H, D)
        return s
    page, lens = case["page"], _lengths(case, gen)
    s["seq_lens"] = lens
    room = -(-(case["hi"] + (T if case["op"] != "decode" else 0)) // page) or 1
    pages = B * room + 1                                   # a page is left over, as there is in a program's pool
    order = torch.randperm(pages, generator=gen, device="cuda")
    s["table"] = order[: B * room].view(B, room).to(torch.int32)
    for name in ("cache_k", "cache_v"):
        s[name] = mk(pages, H, page, D).transpose(1, 2) if case["heads"] else mk(pages, page, H, D)
    if case["op"] == "append":
        s["k"], s["v"] = mk(B, T, H, D), mk(B, T, H, D)
        even = torch.linspace((T + 1) // 2, T, B, dtype=torch.float64).floor().to(torch.int32).cuda()
        s["lengths"] = even[torch.randperm(B, generator=gen, device="cuda")]
        return s
    s["q"] = mk(B, G, H, D)
    if L:
        s["depth_k"], s["depth_v"] = mk(B, L, H, D), mk(B, L, H, D)
    if case["op"] == "step":
        s["k"], s["v"] = mk(B, 1, H, D), mk(B, 1, H, D)
    return s


# ---------------------------------------------------------------- the plain form
def _cos_sin(positions, inv_freq, factor):
    angle = positions.double().unsqueeze(-1) * inv_freq      # 64 bits: far positions
    return (angle.cos() * factor).float(), (angle.sin() * factor).float()


def _rotate(x, cos, sin, case):
    """x [..., D] in 32 bits; cos, sin with a pair's value in the last dimension, broadcast against x."""
    rot = case["rot"]
    if case["pairs"] == "half":
        a, b = x[..., : rot // 2], x[..., rot // 2 : rot]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., rot:]], -1)
    a, b = x[..., 0:rot:2], x[..., 1:rot:2]
    return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), x[..., rot:]], -1)


def _rotate_rows(x, positions, s, inverse=False):
    """x [B, T * G, H, D], row t * G + g at positions[., t]."""
    case = s["case"]
    cos, sin = _cos_sin(positions, s["inv_freq"], s["factor"])           # [B or 1, T, pairs]
    cos, sin = cos[:, :, None, None], (-sin if inverse else sin)[:, :, None, None]
    y = _rotate(x.float().view(x.shape[0], cos.shape[1], -1, *x.shape[2:]), cos, sin, case)
    return y.view(x.shape).to(x.dtype)


def _plain_rotary(s):
    case = s["case"]
    positions = s["positions"] if case["far"] else torch.arange(case["T"], device="cuda")[None]
    out = [_rotate_rows(s[n].detach(), positions, s) for n in ("q", "k")]
    if case["train"]:
        out += [_rotate_rows(s[n], positions, s, inverse=True) for n in ("dq", "dk")]
    return out


def _plain_append(s, lengths):
    case, page = s["case"], s["case"]["page"]
    B, T = s["k"].shape[:2]
    step = torch.arange(T, device="cuda")
    valid = step < lengths[:, None]                                       # [B, T]
    at = s["seq_lens"][:, None] + step
    rows = [torch.where(valid[..., None, None], x, x[:, :1]) for x in (_rotate_rows(s["k"], at, s), s["v"])]
    at = torch.where(valid, at, at[:, :1])                                # tokens behind a prompt's end: its first one again
    pages, slots = s["table"].gather(1, at // page).long(), at % page
    s["cache_k"].index_put_((pages, slots), rows[0])
    s["cache_v"].index_put_((pages, slots), rows[1])


def _plain_decode(s):
    case = s["case"]
    B, H, G, D, L = (case[x] for x in "BHGDL")
    lens = s["seq_lens"].long()
    q = s["q"].float()
    if case["op"] == "step":
        _plain_append(s, torch.ones_like(s["seq_lens"]))
        cos, sin = _cos_sin(lens[:, None, None], s["inv_freq"], s["factor"])
        q = _rotate(q, cos, sin, case)
        lens = lens + 1
    q = q.transpose(1, 2)                                                 # [B, H, G, D]
    keys, values = (s[n][s["table"].long()].flatten(1, 2).float() for n in ("cache_k", "cache_v"))
    visible = torch.arange(keys.shape[1], device="cuda") < lens[:, None]
    if L:
        keys, values = (torch.cat([x, s[n].float()], 1) for x, n in ((keys, "depth_k"), (values, "depth_v")))
        visible = torch.cat([visible, visible.new_ones(B, L)], 1)
    visible = visible[:, None, None]
    score = (q @ keys.permute(0, 2, 3, 1)) * (D ** -0.5)
    score = torch.where(visible, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)                         # a row that sees nothing: o = 0, lse = -inf
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    o = (p @ values.transpose(1, 2)) / torch.where(total == 0, 1.0, total)
    lse = (top + torch.log(total)).squeeze(-1) / math.log(2)
    return o.transpose(1, 2).to(s["q"].dtype), lse.transpose(1, 2).contiguous()


# ---------------------------------------------------------------- the calls of a user
def _own(s):
    import moda_b200 as M
    case = s["case"]
    rotary = M.Rotary(s["inv_freq"], interleaved=case["pairs"] == "interleaved", scale=s["factor"])
    if case["op"] == "rotary":
        q, k = M.rotary_embedding(s["q"], s["k"], rotary, positions=s.get("positions"), moda_group_num=case["G"])
        if not case["train"]:
            return [q, k]
        return [q.detach(), k.detach(), *torch.autograd.grad([q, k], [s["q"], s["k"]], [s["dq"], s["dk"]])]
    cache = (s["cache_k"], s["cache_v"], s["table"], s["seq_lens"])
    if case["op"] == "append":
        M.paged_moda_append(s["k"], s["v"], *cache, lengths=s["lengths"], rotary=rotary)
        return [s["cache_k"], s["cache_v"]]
    depth = dict(cached_k=s.get("depth_k"), cached_v=s.get("depth_v"))
    if case["op"] == "decode":
        return list(M.paged_moda_decode(s["q"], *cache, **depth, moda_group_num=case["G"], need_lse=True))
    o, lse = M.paged_moda_decode(s["q"], *cache, k=s["k"], v=s["v"], **depth, moda_group_num=case["G"], rotary=rotary, need_lse=True)
    return [o, lse, s["cache_k"], s["cache_v"]]


def run(state):
    if own:
        return _own(state)
    case = state["case"]
    if case["op"] == "rotary":
        return _plain_rotary(state)
    if case["op"] == "append":
        _plain_append(state, state["lengths"])
        return [state["cache_k"], state["cache_v"]]
    o, lse = _plain_decode(state)
    return [o, lse] + ([state["cache_k"], state["cache_v"]] if case["op"] == "step" else [])


def _length_sum(case):
    return int(torch.linspace(case["lo"], case["hi"], case["B"], dtype=torch.float64).floor().sum())


def work(case):
    """Bytes: every input read once, every output written once.  Flops: 6 for a rotated pair, 4 D for a query and a
    key that it sees."""
    B, T, H, G, D, L = (case[x] for x in "BTHGDL")
    row = H * D * 2                                        # one token's K (or V), or one of G parts of its q
    if case["op"] == "rotary":
        rows = B * T * (G + 1) * (2 if case["train"] else 1)
        return {"bytes": 2 * rows * row, "flops": 3 * rows * H * case["rot"]}
    if case["op"] == "append":
        tokens = int(torch.linspace((T + 1) // 2, T, B, dtype=torch.float64).floor().sum())
        return {"bytes": 4 * tokens * row, "flops": 3 * tokens * H * case["rot"]}
    keys = _length_sum(case) + B * L
    more = 4 * B * row if case["op"] == "step" else 0      # k and v read, and written to the cache
    own_key = B if case["op"] == "step" else 0
    return {"bytes": 2 * keys * row + 2 * B * G * row + B * G * H * 4 + more, "flops": 4 * D * H * G * (keys + own_key)}


# ---------------------------------------------------------------- from the definition, in 64 bits
def _turned(x, position, case, inv_freq, factor):
    """Rows of x [..., D] (64 bits) as complex numbers turned by their position's angles; position broadcasts against x[..., 0]."""
    rot = case["rot"]
    turn = torch.polar(torch.full_like(inv_freq, factor), torch.zeros_like(inv_freq)) * torch.exp(1j * (position.double()[..., None] * inv_freq))
    y = x.clone()
    if case["pairs"] == "half":
        z = torch.complex(x[..., : rot // 2].contiguous(), x[..., rot // 2 : rot].contiguous()) * turn
        y[..., : rot // 2], y[..., rot // 2 : rot] = z.real, z.imag
    else:
        z = torch.view_as_complex(x[..., :rot].reshape(*x.shape[:-1], rot // 2, 2).contiguous()) * turn
        y[..., :rot] = torch.view_as_real(z).flatten(-2)
    return y


def exact(case, seed):
    s = prepare(case, seed)
    B, T, H, G, D, L = (case[x] for x in "BTHGDL")
    f, factor = s["inv_freq"], s["factor"]
    if case["op"] == "rotary":
        start = s["positions"] if case["far"] else torch.arange(T, device="cuda").expand(B, T)
        out = [torch.empty(s[n].shape, dtype=torch.float64, device="cuda") for n in (("q", "k", "dq", "dk") if case["train"] else ("q", "k"))]
        for y, n in zip(out, ("q", "k", "dq", "dk")):
            for b in range(B):
                groups = s[n].shape[1] // T
                at = start[b].repeat_interleave(groups)[:, None]
                y[b] = _turned(s[n][b].detach().double(), at if n in ("q", "k") else -at, case, f, factor)
        return out
    page, lens = case["page"], s["seq_lens"].tolist()
    more = s["lengths"].tolist() if case["op"] == "append" else [1] * B if case["op"] == "step" else []
    if more:                                               # what the cache holds is held in its type
        for b in range(B):
            at = lens[b] + torch.arange(more[b], device="cuda")
            where, slot = s["table"][b].long()[at // page], at % page
            s["cache_k"][where, slot] = _turned(s["k"][b, : more[b]].double(), at[:, None], case, f, factor).to(s["k"].dtype)
            s["cache_v"][where, slot] = s["v"][b, : more[b]]
    if case["op"] == "append":
        return [s["cache_k"], s["cache_v"]]
    o = torch.zeros(B, G, H, D, dtype=torch.float64, device="cuda")
    lse = torch.full((B, G, H), -math.inf, dtype=torch.float64, device="cuda")
    for b in range(B):
        n = lens[b] + (1 if case["op"] == "step" else 0)
        at = torch.arange(n, device="cuda")
        where, slot = s["table"][b].long()[at // page], at % page
        q = s["q"][b].double()
        if case["op"] == "step":
            q = _turned(q, torch.tensor(n - 1, device="cuda"), case, f, factor)
        keys, values = s["cache_k"][where, slot].double(), s["cache_v"][where, slot].double()
        if L:
            keys, values = torch.cat([keys, s["depth_k"][b].double()]), torch.cat([values, s["depth_v"][b].double()])
        if keys.shape[0] == 0:
            continue
        score = torch.einsum("ghd,nhd->ghn", q, keys) / math.sqrt(D)
        lse[b] = torch.logsumexp(score, -1) / math.log(2)
        o[b] = torch.einsum("ghn,nhd->ghd", torch.softmax(score, -1), values)
    return [o, lse] + ([s["cache_k"], s["cache_v"]] if case["op"] == "step" else [])
