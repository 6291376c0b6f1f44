"""More operators that a training or serving program calls beside the
optimizer's step, as cases that can be timed.

  orth  matrix updates made orthogonal by Newton-Schulz products: X = G / |G|,
        then ``STEPS`` times X <- a X + (b A + c A A) X with A = X X^T (on a
        matrix's smaller side);
  muon  one step of the optimiser that is built on it, for all matrices of a
        model: momentum, orthogonalisation, weight decay and the update;
  qkr   the norm of every head's query and key with the rotation by the token's
        position: the forward pass alone (serving) or with its backward pass.

With ``own`` false the operators run in their plain form, elementary torch
operations in 32 bits, rounded once at the end; with it true through
``scao_amd``.  Everything is made on the GPU from the seed.
"""

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
STEPS, COEFFICIENTS, NORM_EPS = 5, (3.4445, -4.7750, 2.0315), 1e-7
LR, WEIGHT_DECAY, MOMENTUM = 0.02, 0.1, 0.95
HEAD_EPS, ROTARY_BASE = 1e-6, 500000.0


def listed():
    return [
        # a single small matrix, as a probe or an adapter has: launches and host work
        dict(name="orth 256x256 bf16", kind="orth", shapes="256x256*1", dtype="bf16"),
        # the query and output projections of four Llama-1B layers, stacked
        dict(name="orth 8 of 2048x2048 bf16", kind="orth", shapes="2048x2048*8", dtype="bf16"),
        # the largest matrix of the benchmark's models, a Llama-8B layer's gate projection
        dict(name="orth 14336x4096 bf16", kind="orth", shapes="14336x4096*1", dtype="bf16"),
        # matrices of sizes that nothing divides, wide and tall, in the
        # optimizer's default type, as a list
        dict(name="orth odd fp32", kind="orth", shapes="1001x333*12,333x1001*5,77x2049*7",
             dtype="fp32"),
        # the smallest model: a handful of matrices
        dict(name="muon few small fp32", kind="muon", shapes="96x160*1,160x96*1,50x333*2",
             dtype="fp32", nesterov=True),
        # GPT-2-small's attention in fp32
        dict(name="muon gpt2 attention fp32", kind="muon", shapes="768x2304*12,768x768*12",
             dtype="fp32", nesterov=True),
        # four layers of the benchmark's headline model in bf16
        dict(name="muon llama1b layers bf16", kind="muon",
             shapes="2048x2048*8,512x2048*8,8192x2048*8,2048x8192*4", dtype="bf16",
             nesterov=True),
        # serving: one token of one sequence, Llama-8B's heads, far into its context
        dict(name="qkr 1 token llama8b", kind="qkr", train=False, batch=1, seq=1, hq=32, hk=8,
             dim=128, rot=128, far=100000, dtype="bf16", packed=True, interleaved=False),
        # serving: 96 sequences, one token each, every one at a place of its own, Llama-1B's heads
        dict(name="qkr 96 tokens llama1b", kind="qkr", train=False, batch=96, seq=1, hq=32, hk=8,
             dim=64, rot=64, far=16384, dtype="fp16", packed=False, interleaved=False),
        # serving: the prompt of one request, Qwen-3B's heads
        dict(name="qkr 777 tokens qwen3b", kind="qkr", train=False, batch=1, seq=777, hq=16, hk=2,
             dim=128, rot=128, far=0, dtype="bf16", packed=True, interleaved=False),
        # training: four sequences of 2048 tokens, Llama-8B's heads, queries and
        # keys as slices of one projection's rows
        dict(name="qkr train llama8b", kind="qkr", train=True, batch=4, seq=2048, hq=32, hk=8,
             dim=128, rot=128, far=0, dtype="bf16", packed=True, interleaved=False),
        # training in fp32 with odd counts, heads that rotate in part, pairs side by side
        dict(name="qkr train odd fp32", kind="qkr", train=True, batch=3, seq=501, hq=5, hk=3,
             dim=90, rot=34, far=0, dtype="fp32", packed=True, interleaved=True),
    ]


# ------------------------------------------------------------------ draw ---

def _size(rng, lo, hi):
    """A size between lo and hi, spread over its logarithm; half of them whole
    multiples of 64, the others whatever comes, odd ones among them."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5 and v >= 64:
        v = v // 64 * 64
    return max(lo, min(hi, v))


def _products(m, n):
    s, l = min(m, n), max(m, n)
    return STEPS * s * s * (3.0 * l + s)


def draw(rng):
    kind = rng.choice(["orth", "muon", "qkr", "qkr"])
    if kind == "qkr":
        train = rng.random() < 0.5
        seq = _size(rng, 1, 4096) if train else rng.choice([1, _size(rng, 1, 4096)])
        batch = _size(rng, 1, max(1, min(256, 8192 // seq)))
        dim = rng.choice([64, 128, 128, 256, 2 * rng.randint(16, 128)])
        rot = rng.choice([dim, dim, dim, dim // 4 * 2])
        return dict(kind=kind, train=train, batch=batch, seq=seq, hq=rng.choice([4, 12, 16, 32, 7]),
                    hk=rng.choice([1, 2, 4, 8, 3]), dim=dim, rot=rot,
                    far=rng.choice([0, 0, 4096, 120000]),
                    dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                    packed=rng.random() < 0.5, interleaved=rng.random() < 0.3)
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    left = _products(14336, 4096) / (4 if dtype == "fp32" else 1)
    shapes = []
    for _ in range(rng.randint(1, 4)):
        m, n, many = _size(rng, 16, 8192), _size(rng, 16, 8192), rng.choice([1, 1, 4, 16])
        if _products(m, n) * many <= left and m * n * many <= 1 << 28:
            shapes.append("%dx%d*%d" % (m, n, many))
            left -= _products(m, n) * many
    shapes.append("%dx%d*%d" % (_size(rng, 16, 1024), _size(rng, 16, 1024), rng.choice([1, 3])))
    case = dict(kind=kind, shapes=",".join(shapes), dtype=dtype)
    return dict(case, nesterov=rng.random() < 0.8) if kind == "muon" else case


# ---------------------------------------------------------------- inputs ---

def _groups(case):
    """(m, n, how many) of every group of matrices of one shape"""
    out = []
    for part in case["shapes"].split(","):
        shape, many = part.split("*")
        out.append((*(int(x) for x in shape.split("x")), int(many)))
    return out


def _gradients(g, m, n, many, std):
    """Gradients of a layer's weight: noise, and a few directions that stand out
    of it."""
    rank = min(4, m, n)
    strong = torch.randn(many, m, rank, generator=g, device=DEV) @ torch.randn(
        many, rank, n, generator=g, device=DEV)
    noise = torch.randn(many, m, n, generator=g, device=DEV)
    return (noise + strong * ((m + n) / (m * n)) ** 0.5) * std


def _orth_inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [_gradients(g, *shape, 1e-3).to(DTYPES[case["dtype"]]) for shape in _groups(case)]


def _muon_inputs(case, seed):
    """Of every group of one shape, stacked: parameters, their gradients (both of
    the case's type) and the momentum in 32 bits."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt, out = DTYPES[case["dtype"]], []
    for m, n, many in _groups(case):
        p = (torch.randn(many, m, n, generator=g, device=DEV) * n ** -0.5).to(dt)
        grad = _gradients(g, m, n, many, 1e-3).to(dt)
        out.append((p, grad, _gradients(g, m, n, many, 7e-4)))
    return out


def _table(case):
    """Cosines and sines of every position, as a program makes them once."""
    half = case["rot"] // 2
    freq = ROTARY_BASE ** (-torch.arange(half, device=DEV, dtype=torch.float64) / max(half, 1))
    at = torch.arange(case["seq"] + case["far"], device=DEV, dtype=torch.float64)
    angle = at[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def _qkr_inputs(case, seed):
    """Queries and keys as the projections leave them (``packed``: slices of the
    rows of one buffer that also holds the values), weights near one, positions
    that start anywhere, and the gradients of both outputs."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    b, t, hq, hk, dim, dt = (case[k] for k in ("batch", "seq", "hq", "hk", "dim", "dtype"))
    dt = DTYPES[dt]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    if case["packed"]:
        rows = (normal(b, t, (hq + 2 * hk) * dim) * 1.5).to(dt)
        q = rows[..., :hq * dim].unflatten(-1, (hq, dim))
        k = rows[..., hq * dim:(hq + hk) * dim].unflatten(-1, (hk, dim))
    else:
        q, k = ((normal(b, t, h, dim) * 1.5).to(dt) for h in (hq, hk))
    wq, wk = ((1 + 0.2 * normal(dim)).to(dt) for _ in range(2))
    first = torch.randint(0, case["far"] + 1, (b, 1), generator=g, device=DEV)
    positions = first + torch.arange(t, device=DEV)
    return q, k, wq, wk, positions, normal(b, t, hq, dim).to(dt), normal(b, t, hk, dim).to(dt)


def prepare(case, seed):
    if case["kind"] == "orth":
        stacks = _orth_inputs(case, seed)
        return dict(case=case, stacks=stacks, updates=[m for s in stacks for m in s.unbind()])
    if case["kind"] == "muon":
        stacks = _muon_inputs(case, seed)
        state = dict(case=case, stacks=stacks)
        params = []
        for p, grad, buf in stacks:
            for one, its, momentum in zip(p.unbind(), grad.unbind(), buf.unbind()):
                params.append((torch.nn.Parameter(one), momentum))
                params[-1][0].grad = its
        if own:
            import scao_amd
            state["opt"] = opt = scao_amd.Muon(
                [p for p, _ in params], lr=LR, weight_decay=WEIGHT_DECAY, momentum=MOMENTUM,
                nesterov=case["nesterov"], ns_coefficients=COEFFICIENTS, ns_steps=STEPS,
                eps=NORM_EPS)
            for p, momentum in params:
                opt.state[p]["momentum_buffer"] = momentum
        return state
    q, k, wq, wk, positions, dq, dk = _qkr_inputs(case, seed)
    if case["train"]:
        q, k, wq, wk = (t.detach().requires_grad_() for t in (q, k, wq, wk))
    cos, sin = _table(case)
    return dict(case=case, q=q, k=k, wq=wq, wk=wk, positions=positions, dq=dq, dk=dk, cos=cos,
                sin=sin)


# ------------------------------------------------------------------- run ---

def _newton_schulz(x):
    """A stack of matrices in 32 bits, orthogonalised."""
    a, b, c = COEFFICIENTS
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + NORM_EPS)
    for _ in range(STEPS):
        gram = x @ x.mT
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.mT if tall else x


def _plain_muon(state):
    case, out = state["case"], []
    for p, grad, buf in state["stacks"]:
        g = grad.float()
        buf.mul_(MOMENTUM).add_(g * (1 - MOMENTUM))
        update = _newton_schulz(g * (1 - MOMENTUM) + buf * MOMENTUM if case["nesterov"] else buf)
        rate = LR * math.sqrt(max(1.0, p.shape[-2] / p.shape[-1]))
        p.copy_(p.float() * (1 - LR * WEIGHT_DECAY) - rate * update)
        out.append((p, buf))
    return out


def _rotate(y, cos, sin, interleaved, back=False):
    """The first 2 cos.shape[-1] columns of y rotated in pairs (element i with
    element i + half, or 2i with 2i + 1)."""
    half = cos.shape[-1]
    if back:
        sin = -sin
    first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (
        slice(0, half), slice(half, 2 * half))
    out = y.clone()
    out[..., first] = y[..., first] * cos - y[..., second] * sin
    out[..., second] = y[..., second] * cos + y[..., first] * sin
    return out


def _plain_qkr(state):
    case, dt = state["case"], state["q"].dtype
    with torch.no_grad():
        cos, sin = (state[n][state["positions"]][..., None, :] for n in ("cos", "sin"))

        def norm(x, w):
            r = torch.rsqrt(x.square().mean(-1, keepdim=True) + HEAD_EPS)
            return x * r, r, _rotate(x * r * w, cos, sin, case["interleaved"])

        def gradients(dy, unit, r, w):
            dy = _rotate(dy, cos, sin, case["interleaved"], back=True)
            du = dy * w
            return r * (du - unit * (du * unit).mean(-1, keepdim=True)), (dy * unit).sum((0, 1, 2))

        q, k, wq, wk = (state[n].float() for n in ("q", "k", "wq", "wk"))
        uq, rq, yq = norm(q, wq)
        uk, rk, yk = norm(k, wk)
        out = dict(q=yq.to(dt), k=yk.to(dt))
        if case["train"]:
            dq, dwq = gradients(state["dq"].float(), uq, rq, wq)
            dk, dwk = gradients(state["dk"].float(), uk, rk, wk)
            out.update(dq=dq.to(dt), dk=dk.to(dt), dwq=dwq.to(dt), dwk=dwk.to(dt))
    return out


def run(state):
    case = state["case"]
    if case["kind"] == "orth":
        if own:
            import scao_amd
            return scao_amd.orthogonalize(state["updates"], steps=STEPS,
                                          coefficients=COEFFICIENTS, eps=NORM_EPS)
        return [m for s in state["stacks"] for m in _newton_schulz(s.float()).to(s.dtype).unbind()]
    if case["kind"] == "muon":
        if own:
            state["opt"].step()
            return [(p, buf) for p, _, buf in state["stacks"]]
        return _plain_muon(state)
    if not own:
        return _plain_qkr(state)
    import scao_amd
    leaves = [state[n] for n in ("q", "k", "wq", "wk")]
    yq, yk = scao_amd.qk_norm_rope(*leaves, state["cos"], state["sin"], state["positions"],
                                   eps=HEAD_EPS, interleaved=case["interleaved"])
    if not case["train"]:
        return dict(q=yq, k=yk)
    dq, dk, dwq, dwk = torch.autograd.grad((yq, yk), leaves, (state["dq"], state["dk"]))
    return dict(q=yq.detach(), k=yk.detach(), dq=dq, dk=dk, dwq=dwq, dwk=dwk)


# ------------------------------------------------------------------ work ---

def work(case):
    """orth: every matrix read and written once; the products of STEPS steps,
    symmetric ones counted once a pair.  muon: parameter and momentum read and
    written, the gradient read.  qkr: queries and keys read and written, with a
    backward pass their gradients too (inputs and outputs' gradients read,
    gradients written); a table row a token."""
    size = DTYPES[case["dtype"]].itemsize
    if case["kind"] == "qkr":
        tokens = case["batch"] * case["seq"]
        values = tokens * (case["hq"] + case["hk"]) * case["dim"]
        return dict(bytes=values * size * (5 if case["train"] else 2) + tokens * case["rot"] * 4,
                    flops=values * (25.0 if case["train"] else 8.0))
    values = sum(m * n * many for m, n, many in _groups(case))
    flops = sum(_products(m, n) * many for m, n, many in _groups(case))
    return dict(bytes=values * (3 * size + 8 if case["kind"] == "muon" else 2 * size), flops=flops)


# ----------------------------------------------------------------- exact ---

def _exact_orth(g):
    """The factor Q with X = Q G / |G| (or G Q / |G|), a polynomial in the Gram
    matrix of the smaller side, gathered over the steps."""
    a, b, c = COEFFICIENTS
    wide = g.shape[-2] <= g.shape[-1]
    scaled = g / (torch.linalg.matrix_norm(g, keepdim=True) + NORM_EPS)
    gram = torch.matmul(scaled, scaled.mT) if wide else torch.matmul(scaled.mT, scaled)
    eye = torch.eye(gram.shape[-1], dtype=g.dtype, device=g.device).expand_as(gram)
    total = eye
    for _ in range(STEPS):
        factor = a * eye + b * gram + c * torch.matmul(gram, gram)
        total = torch.matmul(factor, total)
        gram = torch.matmul(factor, torch.matmul(gram, factor))
    return torch.matmul(total, scaled) if wide else torch.matmul(scaled, total)


def exact(case, seed):
    """The definitions in 64 bits; the gradients by automatic differentiation,
    the rotation as a product of complex numbers."""
    if case["kind"] == "orth":
        return [m for s in _orth_inputs(case, seed) for m in _exact_orth(s.double()).unbind()]
    if case["kind"] == "muon":
        out = []
        for p, grad, buf in _muon_inputs(case, seed):
            buf = torch.lerp(buf.double(), grad.double(), 1 - MOMENTUM)
            update = torch.lerp(grad.double(), buf, MOMENTUM) if case["nesterov"] else buf
            ratio = max(1.0, p.shape[-2] / p.shape[-1]) ** 0.5
            p = p.double()
            out.append((p - LR * (WEIGHT_DECAY * p + ratio * _exact_orth(update)), buf))
        return out
    q, k, wq, wk, positions, dq, dk = _qkr_inputs(case, seed)
    half = case["rot"] // 2
    freq = torch.pow(torch.tensor(ROTARY_BASE, dtype=torch.float64, device=DEV),
                     -torch.arange(half, dtype=torch.float64, device=DEV) / max(half, 1))
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV),
                       positions[..., None, None] * freq)

    def rotated(x, w):
        y = torch.nn.functional.rms_norm(x, x.shape[-1:], eps=HEAD_EPS) * w
        head, rest = y[..., :2 * half], y[..., 2 * half:]
        pairs = head.unflatten(-1, (half, 2)) if case["interleaved"] else head.unflatten(
            -1, (2, half)).mT
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        z = z if case["interleaved"] else z.mT
        return torch.cat([z.flatten(-2), rest], -1)

    leaves = [t.double().requires_grad_(case["train"]) for t in (q, k, wq, wk)]
    yq, yk = rotated(leaves[0], leaves[2]), rotated(leaves[1], leaves[3])
    if not case["train"]:
        return dict(q=yq, k=yk)
    gq, gk, gwq, gwk = torch.autograd.grad((yq, yk), leaves, (dq.double(), dk.double()))
    return dict(q=yq.detach(), k=yk.detach(), dq=gq, dk=gk, dwq=gwq, dwk=gwk)
