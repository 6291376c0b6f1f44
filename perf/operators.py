"""Operators that a training or serving program calls beside the optimizer's
step, as cases that can be timed.

  ffn   the gated feed-forward block of a decoder layer,
        y = (f(x Wg^T) * (x Wu^T)) Wd^T: the forward pass alone (serving) or
        with its backward pass (training: dx and the three weights' gradients);
  clip  the norm over all gradients of a model and the clipping of the
        gradients to it, between the backward pass and the optimizer's step.

With ``own`` false the operators run in their plain form, elementary torch
operations in 32 bits, rounded once at the end; with it true through
``scao_amd``.  Everything is made on the GPU from the seed.
"""

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
CLIP_EPS = 1e-6

_LLAMA1B = ("128256x2048,2048x2048*32,512x2048*32,8192x2048*32,2048x8192*16,2048*33")
_GPT2 = ("50257x768,768x2304*12,768x768*12,768*50")


def listed():
    return [
        # serving: one token of one sequence through a Llama-1B layer's block.
        # The weights' bytes and the launches
        dict(name="ffn 1 token llama1b", kind="ffn", train=False, tokens=1, d=2048, f=8192,
             dtype="bf16", act="silu", packed=False, pad=0),
        # serving: a batch of 24 sequences, one token each, through a Llama-8B
        # layer's block, gate and up projections in one packed weight
        dict(name="ffn 24 tokens llama8b", kind="ffn", train=False, tokens=24, d=4096, f=14336,
             dtype="bf16", act="silu", packed=True, pad=0),
        # serving: the prompt of one request, no multiple of any tile, through
        # a Qwen-3B layer's block
        dict(name="ffn 777 tokens qwen3b", kind="ffn", train=False, tokens=777, d=2048, f=11008,
             dtype="bf16", act="silu", packed=False, pad=0),
        # training: two sequences of 2048 tokens through a Llama-1B layer's block
        dict(name="ffn train llama1b", kind="ffn", train=True, tokens=4096, d=2048, f=8192,
             dtype="bf16", act="silu", packed=False, pad=0),
        # training: the largest block of the benchmark's models, four sequences
        # of 2048 tokens
        dict(name="ffn train llama8b", kind="ffn", train=True, tokens=8192, d=4096, f=14336,
             dtype="bf16", act="silu", packed=True, pad=0),
        # training in fp16 with sizes that nothing divides and rows that start
        # at any element (the input a slice of wider rows)
        dict(name="ffn train odd fp16", kind="ffn", train=True, tokens=501, d=1001, f=2049,
             dtype="fp16", act="gelu", packed=False, pad=3),
        # training a small model in fp32, the optimizer's default weight type
        dict(name="ffn train gpt2 fp32", kind="ffn", train=True, tokens=2048, d=768, f=2048,
             dtype="fp32", act="gelu_tanh", packed=False, pad=0),
        # the smallest model: a handful of tensors, launches and host work
        dict(name="clip few small fp32", kind="clip", shapes="96x160,160,160x96,96,50x333,1001",
             dtype="fp32", p="2", max_norm=1.0, scale=0.125),
        # GPT-2-small in fp32, gradients summed over eight micro-batches:
        # averaged and clipped in one call
        dict(name="clip gpt2 fp32 mean of 8", kind="clip", shapes=_GPT2, dtype="fp32", p="2",
             max_norm=1.0, scale=0.125),
        # the benchmark's headline model held in bf16
        dict(name="clip llama1b bf16", kind="clip", shapes=_LLAMA1B, dtype="bf16", p="2",
             max_norm=1.0, scale=1.0),
        # adapters and vectors: many odd tensors of two types, largest entry
        dict(name="clip many odd mixed", kind="clip",
             shapes="16x2049*96,1003x8*96,2047*64,1*32,33x65*32,256x128x3x3*12", dtype="mixed",
             p="inf", max_norm=1e-3, scale=0.5),
    ]


# ------------------------------------------------------------------ draw ---

def _size(rng, lo, hi):
    """A size between lo and hi, spread over its logarithm; half of them whole
    multiples of 64, the others whatever comes, odd ones among them."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5 and v >= 64:
        v = v // 64 * 64
    return max(lo, min(hi, v))


def draw(rng):
    if rng.random() < 0.65:
        train = rng.random() < 0.6
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        tokens = _size(rng, 1, 8192)
        d, f = _size(rng, 64, 4096), _size(rng, 128, 14336)
        if dtype == "fp32":   # a sixth of the 16-bit rate
            tokens = min(tokens, 2048)
        return dict(kind="ffn", train=train, tokens=tokens, d=d, f=f, dtype=dtype,
                    act=rng.choice(["silu", "silu", "gelu", "gelu_tanh", "relu", "sigmoid"]),
                    packed=rng.random() < 0.4, pad=rng.choice([0, 0, 0, 1, 64]))
    shapes, left = [], int(math.exp(rng.uniform(math.log(1e4), math.log(4e8))))
    for _ in range(rng.randint(1, 8)):
        m, n, many = _size(rng, 1, 16384), _size(rng, 1, 8192), rng.choice([1, 1, 4, 24])
        if m * n * many <= left:
            shapes.append("%dx%d*%d" % (m, n, many))
            left -= m * n * many
    shapes.append("%d*%d" % (_size(rng, 1, 8192), rng.choice([1, 9, 40])))
    return dict(kind="clip", shapes=",".join(shapes),
                dtype=rng.choice(["fp32", "bf16", "fp16", "mixed"]),
                p=rng.choice(["2", "2", "2", "1", "inf"]), max_norm=rng.choice([0.5, 1.0, 10.0]),
                scale=rng.choice([1.0, 0.25, 0.0625]))


# ---------------------------------------------------------------- inputs ---

def _shapes(case):
    out = []
    for part in case["shapes"].split(","):
        one, _, many = part.partition("*")
        out += [tuple(int(x) for x in one.split("x"))] * int(many or 1)
    return out


def _ffn_inputs(case, seed):
    """x, Wg, Wu, Wd and dy: activations of unit size as a norm layer leaves
    them, weights of a trained layer's size, a loss averaged over the tokens."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    t, d, f, dt = case["tokens"], case["d"], case["f"], DTYPES[case["dtype"]]

    def normal(rows, cols, std):
        return (torch.randn(rows, cols, generator=g, device=DEV) * std).to(dt)

    x = normal(t, d + case["pad"], 1.0)[:, :d]
    if case["packed"]:
        gate, up = normal(2 * f, d, d ** -0.5).split(f)
    else:
        gate, up = normal(f, d, d ** -0.5), normal(f, d, d ** -0.5)
    return x, gate, up, normal(d, f, f ** -0.5), normal(t, d, 0.1)


def _clip_inputs(case, seed):
    """One flat buffer of gradients a type, and the tensors' views of it in
    order, one after the other as gradient buckets hold them.  "mixed": every
    third tensor in bf16, the others in fp32."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    shapes = _shapes(case)
    names = [case["dtype"] if case["dtype"] != "mixed" else "bf16" if i % 3 == 0 else "fp32"
             for i in range(len(shapes))]
    sizes = [math.prod(s) for s in shapes]
    flats, views = {}, {}
    for n in sorted(set(names)):
        total = sum(z for z, m in zip(sizes, names) if m == n)
        flats[n] = (torch.randn(total, generator=g, device=DEV) * 0.01).to(DTYPES[n])
        views[n] = iter(flats[n].split([z for z, m in zip(sizes, names) if m == n]))
    return flats, [next(views[n]).view(s) for n, s in zip(names, shapes)]


def prepare(case, seed):
    if case["kind"] == "ffn":
        x, gate, up, down, dy = _ffn_inputs(case, seed)
        if case["train"]:
            x, gate, up, down = (t.requires_grad_() for t in (x, gate, up, down))
        return dict(case=case, x=x, gate=gate, up=up, down=down, dy=dy)
    flats, grads = _clip_inputs(case, seed)
    params = [torch.nn.Parameter(torch.zeros_like(g)) for g in grads]
    for p, g in zip(params, grads):
        p.grad = g
    return dict(case=case, flats=flats, params=params)


# ------------------------------------------------------------------- run ---

def _act(name, a):
    """f(a) and f'(a)."""
    if name == "silu":
        s = 1 / (1 + torch.exp(-a))
        return a * s, s * (1 + a * (1 - s))
    if name == "sigmoid":
        s = 1 / (1 + torch.exp(-a))
        return s, s * (1 - s)
    if name == "relu":
        on = (a > 0).to(a.dtype)
        return a * on, on
    if name == "gelu":
        cdf = 0.5 * (1 + torch.erf(a * math.sqrt(0.5)))
        return a * cdf, cdf + a * torch.exp(-0.5 * a * a) * (1 / math.sqrt(2 * math.pi))
    c = math.sqrt(2 / math.pi)
    th = torch.tanh(c * (a + 0.044715 * a * a * a))
    return (0.5 * a * (1 + th),
            0.5 * (1 + th) + 0.5 * a * (1 - th * th) * c * (1 + 3 * 0.044715 * a * a))


def _plain_ffn(state):
    case, dt = state["case"], state["x"].dtype
    with torch.no_grad():
        x, gate, up, down = (state[k].float() for k in ("x", "gate", "up", "down"))
        a, b = x @ gate.t(), x @ up.t()
        fa, ga = _act(case["act"], a)
        h = fa * b
        out = dict(y=(h @ down.t()).to(dt))
        if case["train"]:
            dy = state["dy"].float()
            dh = dy @ down
            da, db = dh * b * ga, dh * fa
            out.update(dx=(da @ gate + db @ up).to(dt), dgate=(da.t() @ x).to(dt),
                       dup=(db.t() @ x).to(dt), ddown=(dy.t() @ h).to(dt))
    return out


def _plain_clip(state):
    case = state["case"]
    s, flats = case["scale"], state["flats"]
    wide = {n: f.float() for n, f in flats.items()}
    if case["p"] == "inf":
        norm = torch.stack([w.abs().max() for w in wide.values()]).max() * s
    elif case["p"] == "1":
        norm = torch.stack([w.abs().sum() for w in wide.values()]).sum() * s
    else:
        norm = torch.stack([w.square().sum() for w in wide.values()]).sum().sqrt() * s
    factor = torch.clamp(case["max_norm"] / (norm + CLIP_EPS), max=1.0) * s
    return dict(norm=norm, **{n: flats[n].copy_(w * factor) for n, w in wide.items()})


def run(state):
    case = state["case"]
    if not own:
        return _plain_ffn(state) if case["kind"] == "ffn" else _plain_clip(state)
    import scao_amd
    if case["kind"] == "clip":
        norm = scao_amd.clip_grad_norm_(state["params"], case["max_norm"],
                                        norm_type=float(case["p"]), scale=case["scale"])
        return dict(norm=norm, **state["flats"])
    leaves = [state[k] for k in ("x", "gate", "up", "down")]
    y = scao_amd.gated_ffn(*leaves, activation=case["act"])
    if not case["train"]:
        return dict(y=y)
    dx, dgate, dup, ddown = torch.autograd.grad(y, leaves, state["dy"])
    return dict(y=y.detach(), dx=dx, dgate=dgate, dup=dup, ddown=ddown)


# ------------------------------------------------------------------ work ---

def work(case):
    """The block: inputs and weights read once, outputs and gradients written
    once, three products forward and six backward.  Clipping: the norm reads
    every gradient, the factor needs all of them and then reads and writes
    each."""
    if case["kind"] == "ffn":
        t, d, f, size = case["tokens"], case["d"], case["f"], DTYPES[case["dtype"]].itemsize
        if case["train"]:
            return dict(bytes=size * (4 * t * d + 6 * d * f), flops=18.0 * t * d * f)
        return dict(bytes=size * (2 * t * d + 3 * d * f), flops=6.0 * t * d * f)
    shapes = _shapes(case)
    sizes = [DTYPES[case["dtype"] if case["dtype"] != "mixed" else "bf16" if i % 3 == 0
                    else "fp32"].itemsize for i in range(len(shapes))]
    n = [math.prod(s) for s in shapes]
    return dict(bytes=3 * sum(a * b for a, b in zip(n, sizes)), flops=3.0 * sum(n))


# ----------------------------------------------------------------- exact ---

def _exact_act(name, a):
    if name == "silu":
        return a * torch.sigmoid(a)
    if name == "sigmoid":
        return torch.sigmoid(a)
    if name == "relu":
        return torch.relu(a)
    return torch.nn.functional.gelu(a, approximate="tanh" if name == "gelu_tanh" else "none")


def exact(case, seed):
    """The definitions in 64 bits; the block's gradients by automatic
    differentiation of its forward pass."""
    if case["kind"] == "ffn":
        *leaves, dy = _ffn_inputs(case, seed)
        x, gate, up, down = (t.double().requires_grad_(case["train"]) for t in leaves)
        y = (_exact_act(case["act"], x @ gate.t()) * (x @ up.t())) @ down.t()
        if not case["train"]:
            return dict(y=y)
        dx, dgate, dup, ddown = torch.autograd.grad(y, (x, gate, up, down), dy.double())
        return dict(y=y.detach(), dx=dx, dgate=dgate, dup=dup, ddown=ddown)
    flats, _ = _clip_inputs(case, seed)
    ord_ = float(case["p"])
    parts = torch.stack([torch.linalg.vector_norm(f, ord_, dtype=torch.float64)
                         for f in flats.values()])
    norm = torch.linalg.vector_norm(parts, ord_) * case["scale"]
    factor = case["scale"] * torch.clamp(case["max_norm"] / (norm + CLIP_EPS), max=1.0)
    return dict(norm=norm, **{n: f.double() * factor for n, f in flats.items()})
