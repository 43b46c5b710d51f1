"""Operators of a ragged batch's step as cases: each in plain torch operations and as a user calls it.

  append    the rows of several sequences' new tokens: queries and keys turned to their positions, keys
            and values into paged caches (device.append_batch)
  packed    causal attention of several prompts in one run of rows, some behind a cached prefix
            (device.attention_packed)
  rows8     rows to 8-bit codes with a scale each (device.quantise_rows_int8)
  linear8   such rows through a weight of 8-bit codes (device.linear_int8, linear_int8_accumulate)
  sample    a token of every row of logits by temperature, top-k, top-p and min-p from a given
            uniform number (device.sample, sample_f32)

The models are the three the library names; pages hold 32 positions at FP16.
"""

import math
import sys
from pathlib import Path

import numpy as np
import torch

#: False: run() computes in plain torch operations. True: it calls the library.
own = False

PACKAGE = Path(__file__).resolve().parent.parent / "semantic-aware_adaptive_kv_cache_precision_amd"
P = 32
UNREAD = 255  # the tier of a page that is not there
#: layers' heads, KV heads, head_dim, hidden and FFN widths, vocabulary, RoPE base.
MODELS = {
    "qwen2.5-0.5b": dict(heads=14, kv=2, hd=64, hidden=896, ffn=4864, vocab=151936, theta=1e6),
    "qwen2.5-1.5b": dict(heads=12, kv=2, hd=128, hidden=1536, ffn=8960, vocab=151936, theta=1e6),
    "llama-3.2-1b": dict(heads=32, kv=8, hd=64, hidden=2048, ffn=8192, vocab=128256, theta=5e5),
}
#: Rotary angles scaled for long contexts, as models' configurations give them.
SCALINGS = {
    "none": None,
    "linear": dict(kind="linear", factor=4.0),
    "llama3": dict(kind="llama3", factor=32.0, low=1.0, high=4.0, original=8192),
    "yarn": dict(kind="yarn", factor=4.0, original=32768),
}


def listed():
    return [
        # One new token of each of 32 conversations; the prompts of a few, with scaled angles.
        dict(name="append_32_1.5b", kind="append", model="qwen2.5-1.5b", batch=32, rows=32,
             longest=8192, order=1, scaling="none", part=128, interleaved=False, fused=True),
        dict(name="append_prompts_llama", kind="append", model="llama-3.2-1b", batch=7, rows=9001,
             longest=16640, order=2, scaling="llama3", part=64, interleaved=False, fused=True),
        # A few short chats; long prompts of different lengths; new turns behind cached prefixes.
        dict(name="packed_chats_0.5b", kind="packed", model="qwen2.5-0.5b", batch=9, rows=413,
             past=0, order=3, fused=True),
        dict(name="packed_prompts_1.5b", kind="packed", model="qwen2.5-1.5b", batch=8, rows=12000,
             past=0, order=4, fused=True),
        dict(name="packed_turns_llama", kind="packed", model="llama-3.2-1b", batch=12, rows=3001,
             past=6000, order=5, fused=False),
        # A small batch's rows before a projection; a chunk's before the down projection.
        dict(name="rows8_5_0.5b", kind="rows8", rows=5, inn=896),
        dict(name="rows8_2k_1.5b", kind="rows8", rows=2048, inn=8960),
        # The rows of a batch of tokens; of a chunk through gate; of prompts into the residual.
        dict(name="linear8_24_llama", kind="linear8", rows=24, inn=2048, out=8192, bias=False,
             add=False),
        dict(name="linear8_4k_1.5b", kind="linear8", rows=4096, inn=1536, out=8960, bias=True,
             add=False),
        dict(name="linear8_add_llama", kind="linear8", rows=1777, inn=8192, out=2048, bias=False,
             add=True),
        # One sequence's token; a batch's, each request with settings of its own.
        dict(name="sample_1_llama", kind="sample", model="llama-3.2-1b", rows=1, order=6, half=False,
             settings="all"),
        dict(name="sample_48_qwen", kind="sample", model="qwen2.5-1.5b", rows=48, order=7, half=False,
             settings="mixed"),
    ]


def _spread(rng, low, high):
    """A whole number, spread over the range's logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(("append", "packed", "packed", "rows8", "linear8", "linear8", "sample"))
    if kind == "rows8":
        inn = 16 * _spread(rng, 1, 560)
        return dict(kind=kind, inn=inn, rows=_spread(rng, 1, min(8192, 2048 * 8960 // inn)))
    if kind == "linear8":
        inn, out = 16 * _spread(rng, 1, 560), _spread(rng, 1, 16384)
        return dict(kind=kind, inn=inn, out=out, bias=rng.random() < 0.5, add=rng.random() < 0.3,
                    rows=_spread(rng, 1, min(8192, max(1, 4096 * 8960 * 1536 // (inn * out)))))
    model = rng.choice(sorted(MODELS))
    c = dict(kind=kind, model=model, order=rng.randint(1, 1 << 20))
    if kind == "sample":
        c.update(rows=_spread(rng, 1, 48), half=rng.random() < 0.4,
                 settings=rng.choice(("mixed", "all", "temperature", "top_k", "top_p", "min_p")))
        return c
    c.update(fused=rng.random() < 0.5, batch=_spread(rng, 1, 48))
    if kind == "append":
        s = MODELS[model]
        c.update(rows=rng.choice((c["batch"], _spread(rng, c["batch"], 8192))),
                 scaling=rng.choice(sorted(SCALINGS)), interleaved=rng.random() < 0.4,
                 part=rng.choice((s["hd"], s["hd"], s["hd"] // 2, s["hd"] // 4)))
        c["longest"] = _spread(rng, 64, 32768)
        c["rows"] = min(c["rows"], c["batch"] * c["longest"])
    else:
        c["past"] = rng.choice((0, 0, _spread(rng, 1, 8192)))
        c["batch"] = min(c["batch"], 32768 // (c["past"] + 1) + 1)
        c["rows"] = _spread(rng, c["batch"], 4096 if c["past"] else 8192)
    return c


def _cut(rng, rows, batch, most=None):
    """`batch` whole numbers that make `rows`, some of them nothing, none over `most`."""
    share = rng.exponential(1.0, batch) ** 1.5 * (rng.random(batch) > 0.06)
    share[rng.integers(0, batch)] += 0.3
    n = np.floor(rows * share / share.sum()).astype(np.int64)
    n[np.argmax(n)] += rows - n.sum()
    if most is not None:
        over = np.maximum(n - most, 0).sum()
        n = np.minimum(n, most)
        for i in range(batch):
            more = min(over, most - n[i])
            n[i] += more
            over -= more
    return n


def _counts(c):
    """New tokens and lengths of the sequences, from the case alone."""
    rng = np.random.default_rng(c["order"])
    if c["kind"] == "append" and c["rows"] == c["batch"]:
        n = np.ones(c["batch"], np.int64)
    else:
        n = _cut(rng, c["rows"], c["batch"], c.get("longest"))
    if c["kind"] == "append":
        room = c["longest"] - n
        return n, n + np.floor(rng.random(c["batch"]) * (room + 1)).astype(np.int64)
    if not c["past"]:
        return n, n
    return n, n + rng.integers(0, 2 * c["past"] + 1, c["batch"])


# -- inputs, made from the seed alone ------------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(1 + 7919 * seed)
    return g


def _normal(g, *shape, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).half()


def _wide(g, rows, width):
    """Rows whose channels are N(0, 1), a fiftieth of them ten times larger."""
    x = torch.randn((rows, width), generator=g, device="cuda")
    x[:, torch.randperm(width, generator=g, device="cuda")[:round(width / 50)]] *= 10.0
    return x.half()


def _sequence_inputs(c, seed):
    s, g = MODELS[c["model"]], _generator(seed)
    n, length = _counts(c)
    keys = int(n.sum()) if c["kind"] == "append" else int(length.sum())
    return (s, n, length, _normal(g, int(n.sum()), s["heads"] * s["hd"]),
            _wide(g, keys, s["kv"] * s["hd"]), _normal(g, keys, s["kv"] * s["hd"]))


def _slots(c, seed):
    """Each sequence's pages as places in the pool, in any order."""
    n, length = _counts(c)
    pages = -(-length // P)
    order = np.random.default_rng([seed, 3]).permutation(int(pages.sum()))
    return n, length, np.split(order, np.cumsum(pages)[:-1])


def _linear_inputs(c, seed):
    g = _generator(seed)
    x = _wide(g, c["rows"], c["inn"])
    if c["kind"] == "rows8":
        return x, None, None, None
    w = _normal(g, c["out"], c["inn"], scale=c["inn"] ** -0.5)
    bias = _normal(g, c["out"]) if c["bias"] else None
    y = torch.randn((c["rows"], c["out"]), generator=g, device="cuda") if c["add"] else None
    return x, w, bias, y


def _sample_inputs(c, seed):
    """Logits N(0, 2) with some forty tokens raised, a uniform number a row, and the settings."""
    g, rows, vocab = _generator(seed), c["rows"], MODELS[c["model"]]["vocab"]
    x = 2.0 * torch.randn((rows, vocab), generator=g, device="cuda")
    at = torch.randint(0, vocab, (rows, 40), generator=g, device="cuda")
    x.scatter_add_(1, at, 4.0 * torch.rand((rows, 40), generator=g, device="cuda").log().neg())
    u = torch.rand(rows, generator=g, device="cuda")
    rng = np.random.default_rng(c["order"])
    which = c["settings"]
    t = rng.uniform(0.4, 1.6, rows)
    k = np.round(np.exp(rng.uniform(0, math.log(500), rows)))
    p, m = rng.uniform(0.5, 1.0, rows), rng.uniform(0.0, 0.2, rows)
    if which == "mixed":  # each request has some of them
        t[rng.random(rows) < 0.1] = 0.0
        k[rng.random(rows) < 0.5] = 0
        p[rng.random(rows) < 0.4] = 1.0
        m[rng.random(rows) < 0.5] = 0.0
    on = {name: torch.tensor(v, dtype=d).cuda() for name, v, d in
          (("temperature", t, torch.float32), ("top_k", k, torch.int32),
           ("top_p", p, torch.float32), ("min_p", m, torch.float32))}
    return (x.half() if c["half"] else x), u, {
        name: v for name, v in on.items() if which in ("mixed", "all", name)}


class _On:
    """A torch tensor where the library takes a device tensor: its address, its elements (to the
    end of the memory it is a view of) and their bytes."""

    def __init__(self, tensor, base=None):
        self.tensor, self.base = tensor, tensor if base is None else base
        self.address = tensor.data_ptr()
        self.numel = self.base.numel() - (self.address - self.base.data_ptr()) // tensor.element_size()
        self.nbytes = self.numel * tensor.element_size()


def _empty(*shape, dtype=torch.float16):
    return torch.zeros(shape, dtype=dtype, device="cuda")


def _codes(x):
    """Rows as whole numbers -127 .. 127 and the fp32 scale they are in."""
    top = x.float().abs().amax(1, keepdim=True)
    scale = top / torch.full_like(top, 127.0)  # a division, where a plain number's is a product
    code = torch.round(x.float() / torch.where(scale > 0, scale, 1.0))
    return code.to(torch.int8), scale[:, 0]


def _ints(values):
    return torch.from_numpy(np.asarray(values, np.int32)).cuda()


def prepare(case, seed):
    c = case
    if c["kind"] in ("rows8", "linear8"):
        x, w, bias, y = _linear_inputs(c, seed)
        if c["kind"] == "rows8":
            st = dict(c=c, x=x, codes=_empty(c["rows"], c["inn"], dtype=torch.int8),
                      scales=_empty(c["rows"], dtype=torch.float32))
        else:
            st = dict(c=c, bias=bias, y0=y)
            st["codes"], st["scales"] = _codes(x)
            st["w_codes"], st["w_scales"] = _codes(w)
            st["y"] = _empty(c["rows"], c["out"], dtype=torch.float32 if c["add"] else torch.float16)
    elif c["kind"] == "sample":
        x, u, settings = _sample_inputs(c, seed)
        st = dict(c=c, x=x, u=u, settings=settings, tokens=_empty(c["rows"], dtype=torch.int32))
        st["settings_on"] = {name: _On(v) for name, v in settings.items()}
        if own:  # the memory a serving loop keeps for its steps' choices
            floats = _library().sample_scratch(c["rows"], x.shape[1])
            st["scratch"] = _On(_empty(max(4, floats), dtype=torch.float32))
    else:
        s, n, length, q, k, v = _sequence_inputs(c, seed)
        base = None
        if c["fused"] and len(q) == len(k):
            base = torch.cat([q, k, v], 1)
            q, k, v = base.split([q.shape[1], k.shape[1], v.shape[1]], 1)
        st = dict(c=c, s=s, n=n, length=length, q=q, k=k, v=v)
        st["on"] = [_On(t, base) for t in (q, k, v)]
        st["offsets"] = _ints(np.concatenate([[0], np.cumsum(n)]))
        if c["kind"] == "packed":
            st["out"] = _empty(len(q), s["heads"], s["hd"])
            st["offsets_k"] = _ints(np.concatenate([[0], np.cumsum(length)]))
            # The memory a serving loop keeps for the parts of long ranges that are joined at the end.
            st["parts"] = _On(_empty(1 << 24, dtype=torch.float32))
        else:
            _, _, slots = _slots(c, seed)
            most = max(1, -(-c["longest"] // P))
            st["pool"] = _empty(max(1, sum(map(len, slots))), 2, P, s["kv"] * s["hd"])
            table = np.zeros((c["batch"], most), np.int64)
            tiers = np.full((c["batch"], most), UNREAD, np.uint8)
            for i, places in enumerate(slots):
                table[i, :len(places)] = st["pool"].data_ptr() + places * (4 * P * s["kv"] * s["hd"])
                tiers[i, :len(places)] = 0
            # The place and row of every token in the pool.
            at = [np.arange(e - m, e) for m, e in zip(n, length)]
            st["place"] = torch.from_numpy(np.concatenate(
                [p[t // P] for p, t in zip(slots, at)])).cuda()
            st["position"] = torch.from_numpy(np.concatenate(at)).cuda()
            st.update(pages=torch.from_numpy(table).cuda(), tiers=torch.from_numpy(tiers).cuda(),
                      lengths=_ints(length), q_out=_empty(len(q), s["heads"], s["hd"]),
                      k_out=_empty(len(q), s["kv"], s["hd"]))
            if own:
                st["rope"] = _library().RopeTable(c["part"], s["theta"], scaling=SCALINGS[c["scaling"]])
                st["rope"].cover(P * most)
    for name in ("x", "codes", "scales", "bias", "w_codes", "w_scales", "y", "y0", "u", "tokens", "offsets",
                 "offsets_k", "out", "pages", "tiers", "lengths", "q_out", "k_out"):
        if st.get(name) is not None:
            st[name + "_on"] = _On(st[name])
    return st


# -- one pass --------------------------------------------------------------------------------------

def _library():
    if str(PACKAGE) not in sys.path:
        sys.path.insert(0, str(PACKAGE))
    from microinfer import _microinfer
    return _microinfer.device


def run(state):
    st, c = state, state["c"]
    return globals()[("_own_" if own else "_plain_") + c["kind"]](st, c)


def _own_append(st, c):
    s, (q, k, v) = st["s"], st["on"]
    _library().append_batch(q, k, v, st["q_out_on"], st["k_out_on"], st["pages_on"], st["tiers_on"],
                            st["lengths_on"], st["offsets_on"], c["batch"], st["tiers"].shape[1],
                            len(st["q"]), st["rope"], s["heads"], s["kv"], s["hd"],
                            interleaved=c["interleaved"], q_stride=st["q"].stride(0),
                            k_stride=st["k"].stride(0), v_stride=st["v"].stride(0))
    return st["q_out"], st["k_out"], st["pool"]


def _own_packed(st, c):
    s, (q, k, v) = st["s"], st["on"]
    _library().attention_packed(q, k, v, st["out_on"], st["offsets_on"], st["offsets_k_on"],
                                c["batch"], len(st["q"]), len(st["k"]), s["heads"], s["kv"], s["hd"],
                                q_stride=st["q"].stride(0), k_stride=st["k"].stride(0),
                                v_stride=st["v"].stride(0), partials=st["parts"])
    return st["out"]


def _own_rows8(st, c):
    _library().quantise_rows_int8(st["x_on"], st["codes_on"], st["scales_on"], c["rows"], c["inn"])
    return st["codes"], st["scales"]


def _own_linear8(st, c):
    parts = st["codes_on"], st["scales_on"], st["w_codes_on"], st["w_scales_on"]
    if c["add"]:
        _library().linear_int8_accumulate(*parts, st["y_on"], c["rows"], c["inn"], c["out"],
                                          residual=st["y0_on"])
        return st["y"]
    _library().linear_int8(*parts, st.get("bias_on"), st["y_on"], c["rows"], c["inn"], c["out"])
    return st["y"]


def _own_sample(st, c):
    d = _library()
    (d.sample if c["half"] else d.sample_f32)(st["x_on"], st["u_on"], st["tokens_on"], c["rows"],
                                             st["x"].shape[1], scratch=st["scratch"],
                                             **st["settings_on"])
    return st["tokens"]


def _frequencies(c, theta):
    """The angles a position turns each pair by, and the factor of cos and sin; float64."""
    part, scaling = c["part"], SCALINGS[c["scaling"]]
    f = theta ** (-torch.arange(0, part, 2, device="cuda", dtype=torch.float64) / part)
    if scaling is None:
        return f, 1.0
    factor = scaling["factor"]
    if scaling["kind"] == "linear":
        return f / factor, 1.0
    if scaling["kind"] == "llama3":
        # Turns over the original context: few are slowed whole, many not at all.
        turns = scaling["original"] * f / (2 * math.pi)
        keep = ((turns - scaling["low"]) / (scaling["high"] - scaling["low"])).clamp(0, 1)
        return f * (keep + (1 - keep) / factor), 1.0

    def pair(turns):  # the pair that turns so often over the original context
        return part * math.log(scaling["original"] / (turns * 2 * math.pi)) / (2 * math.log(theta))

    low, high = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), part - 1)
    slow = ((torch.arange(part // 2, device="cuda", dtype=torch.float64) - low) /
            max(high - low, 0.001)).clamp(0, 1)
    return f * (1 - slow + slow / factor), 0.1 * math.log(factor) + 1.0


def _turned(x, position, c, s):
    """Rows (n, heads, hd) turned to their positions: the angles in 64 bits, the rest in x's type."""
    f, magnitude = _frequencies(c, s["theta"])
    angle = position.double()[:, None] * f
    cos, sin = ((t * magnitude).to(x.dtype)[:, None] for t in (angle.cos(), angle.sin()))
    out, half = x.clone(), c["part"] // 2
    a, b = ((slice(0, c["part"], 2), slice(1, c["part"], 2)) if c["interleaved"] else
            (slice(0, half), slice(half, c["part"])))
    out[..., a] = x[..., a] * cos - x[..., b] * sin
    out[..., b] = x[..., b] * cos + x[..., a] * sin
    return out


def _plain_append(st, c):
    s = st["s"]
    q, k = (_turned(st[x].float().reshape(len(st[x]), -1, s["hd"]), st["position"], c, s).half()
            for x in ("q", "k"))
    row = st["position"] % P
    st["pool"][st["place"], 0, row] = k.flatten(1)
    st["pool"][st["place"], 1, row] = st["v"]
    return q, k, st["pool"]


def _plain_packed(st, c):
    s, outs, q0, k0 = st["s"], [], 0, 0
    group = s["heads"] // s["kv"]
    for n, length in zip(st["n"].tolist(), st["length"].tolist()):
        q = st["q"][q0:q0 + n].float().reshape(n, s["kv"], group, s["hd"]).permute(1, 2, 0, 3)
        k, v = (st[x][k0:k0 + length].float().reshape(length, s["kv"], s["hd"]).transpose(0, 1)
                for x in ("k", "v"))
        q0, k0 = q0 + n, k0 + length
        score = (q.reshape(s["kv"], group * n, s["hd"]) * s["hd"] ** -0.5) @ k.transpose(1, 2)
        score = score.reshape(s["kv"], group, n, length)
        hidden = torch.arange(length, device="cuda") > torch.arange(
            length - n, length, device="cuda")[:, None]
        p = score.masked_fill_(hidden, -math.inf)
        if n:
            p = p.sub_(p.amax(3, keepdim=True)).exp_()
        total = p.sum(3, keepdim=True)
        out = (p.reshape(s["kv"], group * n, length) @ v).reshape(s["kv"], group, n, s["hd"]) / total
        outs.append(out.permute(2, 0, 1, 3).reshape(n, s["heads"], s["hd"]).half())
    return torch.cat(outs)


def _plain_rows8(st, c):
    return _codes(st["x"])


def _plain_linear8(st, c):
    y = (st["codes"].float() @ st["w_codes"].float().T) * st["scales"][:, None] * st["w_scales"]
    if c["add"]:
        return st["y0"] + y
    return (y if st["bias"] is None else y + st["bias"].float()).half()


def _plain_sample(st, c):
    x, rows = st["x"].double(), c["rows"]
    get = st["settings"].get
    off = torch.zeros(rows, device="cuda")
    t, k, p, m = (get("temperature", off + 1), get("top_k", off), get("top_p", off + 1),
                  get("min_p", off))
    x, order = torch.sort(x, dim=1, descending=True, stable=True)
    t = t.double()[:, None]
    w = ((x - x[:, :1]) / torch.where(t > 0, t, 1.0)).exp()
    rank = torch.arange(x.shape[1], device="cuda")[None]
    keep = (rank < k[:, None]) | (k[:, None] <= 0)
    keep &= (rank == 0) | (t > 0)
    w = w * keep
    before = w.cumsum(1) - w
    total = w.sum(1, keepdim=True)
    p = p.double()[:, None]
    w = w * ((before < p * total) | (p >= 1) | (rank == 0))
    w = w * (w >= m.double()[:, None])
    w = torch.zeros_like(w).scatter_(1, order, w)
    reach = w.cumsum(1)
    return (reach <= st["u"].double()[:, None] * reach[:, -1:]).sum(1).to(torch.int32)


# -- the work that cannot be done without -----------------------------------------------------------

def work(case):
    c = case
    if c["kind"] == "rows8":
        n = c["rows"] * c["inn"]
        return dict(bytes=3.0 * n + 4 * c["rows"], flops=3.0 * n)
    if c["kind"] == "linear8":
        m, n, k = c["rows"], c["out"], c["inn"]
        return dict(bytes=float(m * k + n * k + 4 * (m + n) + (8 if c["add"] else 2) * m * n +
                                2 * n * c["bias"]), flops=2.0 * m * n * k)
    if c["kind"] == "sample":
        n = c["rows"] * MODELS[c["model"]]["vocab"]
        return dict(bytes=float((2 if c["half"] else 4) * n + 24 * c["rows"]), flops=4.0 * n)
    s = MODELS[c["model"]]
    n, length = _counts(c)
    rows, w = int(n.sum()), s["kv"] * s["hd"]
    if c["kind"] == "append":
        # q read and written, k read and written twice, v read and written, the angles.
        return dict(bytes=float(rows * (4 * s["heads"] * s["hd"] + 10 * w + 4 * c["part"])),
                    flops=3.0 * rows * (s["heads"] + s["kv"]) * c["part"])
    seen = (n * (length - n) + n * (n + 1) / 2).sum()
    return dict(bytes=float(4 * length.sum() * w + 4 * rows * s["heads"] * s["hd"]),
                flops=4.0 * s["heads"] * s["hd"] * float(seen))


# -- what run() returns, in 64 bits -----------------------------------------------------------------

def _exact_angles(c, s, position):
    """cos and sin of position * frequency, times the scaling's factor, (n, pairs) in float64."""
    half, scaling = c["part"] // 2, SCALINGS[c["scaling"]] or dict(kind="none")
    kind, freq, grow = scaling["kind"], [], 1.0
    for j in range(half):
        f = s["theta"] ** (-2.0 * j / c["part"])
        if kind == "linear":
            f /= scaling["factor"]
        elif kind == "llama3":
            wave = 2 * math.pi / f
            if wave > scaling["original"] / scaling["low"]:
                f /= scaling["factor"]
            elif wave >= scaling["original"] / scaling["high"]:
                smooth = (scaling["original"] / wave - scaling["low"]) / (scaling["high"] - scaling["low"])
                f = (1 - smooth) * f / scaling["factor"] + smooth * f
        elif kind == "yarn":
            ends = [c["part"] * math.log(scaling["original"] / (turns * 2 * math.pi)) /
                    (2 * math.log(s["theta"])) for turns in (32.0, 1.0)]
            low, high = max(math.floor(ends[0]), 0), min(math.ceil(ends[1]), c["part"] - 1)
            ramp = min(1.0, max(0.0, (j - low) / max(high - low, 0.001)))
            f = f / scaling["factor"] * ramp + f * (1 - ramp)
            grow = 0.1 * math.log(scaling["factor"]) + 1.0
        freq.append(f)
    angle = np.outer(position.astype(np.float64), np.array(freq))
    return (torch.from_numpy(np.cos(angle) * grow).cuda(), torch.from_numpy(np.sin(angle) * grow).cuda())


def _exact_append(c, seed):
    s, n, length, q, k, v = _sequence_inputs(c, seed)
    _, _, slots = _slots(c, seed)
    position = np.concatenate([np.arange(e - m, e) for m, e in zip(n, length)])
    cos, sin = _exact_angles(c, s, position)
    pairs = torch.arange(c["part"] // 2, device="cuda")
    a, b = (2 * pairs, 2 * pairs + 1) if c["interleaved"] else (pairs, pairs + c["part"] // 2)
    turned = []
    for x in (q, k):
        x = x.double().reshape(len(x), -1, s["hd"])
        y = x.clone()
        turn = torch.complex(x[:, :, a], x[:, :, b]) * torch.complex(cos, sin)[:, None]
        y[:, :, a], y[:, :, b] = turn.real, turn.imag
        turned.append(y)
    pool = torch.zeros(max(1, sum(map(len, slots))), 2, P, s["kv"] * s["hd"], device="cuda",
                       dtype=torch.float64)
    begin = 0
    for m, e, places in zip(n.tolist(), length.tolist(), slots):
        for t in range((e - m) // P * P, e, P):  # a page at a time
            lo, hi = max(t, e - m), min(t + P, e)
            mine = slice(begin + lo - (e - m), begin + hi - (e - m))
            if hi > lo:
                pool[places[t // P], 0, lo - t:hi - t] = turned[1][mine].flatten(1)
                pool[places[t // P], 1, lo - t:hi - t] = v[mine].double()
        begin += m
    return turned[0], turned[1], pool


def _exact_packed(c, seed):
    s, n, length, q, k, v = _sequence_inputs(c, seed)
    group = s["heads"] // s["kv"]
    out = torch.zeros(len(q), s["heads"], s["hd"], device="cuda", dtype=torch.float64)
    q, (k, v) = q.double().reshape(len(q), -1, s["hd"]), (
        x.double().reshape(len(x), s["kv"], s["hd"]) for x in (k, v))
    q0 = k0 = 0
    for m, e in zip(n.tolist(), length.tolist()):
        above = torch.ones(m, e, dtype=torch.bool, device="cuda").triu(e - m + 1)
        for h in range(s["heads"]):
            score = (q[q0:q0 + m, h] @ k[k0:k0 + e, h // group].T / math.sqrt(s["hd"]))
            out[q0:q0 + m, h] = torch.softmax(score.masked_fill_(above, -math.inf), 1) @ v[k0:k0 + e, h // group]
        q0, k0 = q0 + m, k0 + e
    return out


def _exact_codes(x):
    """Codes by the rule (a division in 32 bits, to the nearest, even at halves), and the scale."""
    scale = (x.double().abs().amax(1) / 127.0).float()
    q = x.float() / torch.where(scale == 0, torch.ones_like(scale), scale)[:, None]
    return q.double().round(), scale


def _exact_sample(c, seed):
    x, u, settings = _sample_inputs(c, seed)
    x, u = x.cpu().numpy().astype(np.float64), u.cpu().numpy().astype(np.float64)
    settings = {name: v.cpu().numpy().astype(np.float64) for name, v in settings.items()}
    tokens = []
    for i, row in enumerate(x):
        t, k, p, m = (settings[name][i] if name in settings else default for name, default in
                      (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0)))
        if t <= 0:
            tokens.append(int(np.argmax(row)))
            continue
        order = np.argsort(-row, kind="stable")
        if k > 0:
            order = order[:int(k)]
        w = np.exp((row[order] - row[order[0]]) / t)
        if p < 1:
            reach = np.cumsum(w)
            w = w[:max(1, int(np.searchsorted(reach, p * reach[-1], side="left")) + 1)]
        w = w[w >= m]
        order = order[:len(w)]
        by_index = np.argsort(order)
        reach = np.cumsum(w[by_index])
        tokens.append(int(order[by_index][np.searchsorted(reach, u[i] * reach[-1], side="right")]))
    return torch.tensor(tokens, dtype=torch.int32)


def exact(case, seed):
    c = case
    if c["kind"] == "append":
        return _exact_append(c, seed)
    if c["kind"] == "packed":
        return _exact_packed(c, seed)
    if c["kind"] == "sample":
        return _exact_sample(c, seed)
    x, w, bias, y = _linear_inputs(c, seed)
    code, scale = _exact_codes(x)
    if c["kind"] == "rows8":
        return code.to(torch.int8), scale.double()
    w_code, w_scale = _exact_codes(w)
    out = (code @ w_code.T) * torch.outer(scale.double(), w_scale.double())
    if y is not None:
        return y.double() + out
    return out if bias is None else out + bias.double()
