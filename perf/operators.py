"""Cases, inputs and plain forms of the training-step operators: log-probabilities of given classes (with entropy and top
alternatives, and their gradient), orthogonalisation of updates by Newton-Schulz products, and the Muon update built on it.

With `own` false run() computes the formulas with elementary torch operations in 32 bits, rounded once at the end; with
`own` true it makes the calls of gmc.classification and gmc.optimisation."""
import math
import os
import sys

import torch

own = False

PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gaussian-mixture-convolution-networks_b200")
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
IGNORED = -100
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS = 5
EPSILON = 1e-7


def log_probs_case(name, rows, classes, dtype, n_top, train, temperature=1.0, masked=0.0):
    return {"name": name, "op": "log_probabilities", "rows": rows, "classes": classes, "dtype": dtype, "n_top": n_top,
            "train": train, "temperature": temperature, "masked": masked}


def orthogonalise_case(name, batch, rows, cols, dtype):
    return {"name": name, "op": "orthogonalise", "batch": batch, "rows": rows, "cols": cols, "dtype": dtype}


def muon_case(name, shapes, dtype, nesterov=True):
    return {"name": name, "op": "muon", "shapes": shapes, "dtype": dtype, "nesterov": nesterov}


def listed():
    return [
        # one mixture classified into the ten classes of the default network, the five likeliest with it: latency
        log_probs_case("ten classes one sample", 1, 10, "float32", 5, False),
        # a training step of the classifier on forty classes: the loss, its entropy term and the gradient
        log_probs_case("forty classes training", 256, 40, "float32", 0, True),
        # one generated token over a mid-size odd vocabulary with twenty alternatives, at a sampling temperature
        log_probs_case("one token of 50257", 1, 50257, "bfloat16", 20, False, temperature=0.7),
        # a decoding batch over a large vocabulary whose last entries are padding (masked out)
        log_probs_case("64 tokens of 131072", 64, 131072, "bfloat16", 8, False, masked=0.01),
        # a language-model training step in 16 bits, ragged in both directions
        log_probs_case("training 4093x32003", 4093, 32003, "bfloat16", 0, True),
        # the same in 32 bits over a large odd vocabulary, with the top alternatives' gradient (distillation)
        log_probs_case("training 1021x100003", 1021, 100003, "float32", 4, True, masked=0.05),
        # the kernel weights of the network's deepest layer, 64 x (32 channels * 5 components)
        orthogonalise_case("layer weights 64x160", 1, 64, 160, "float32"),
        # a stack of projection matrices of one shape, taller than wide
        orthogonalise_case("24 projections 1024x256", 24, 1024, 256, "bfloat16"),
        # a square hidden matrix
        orthogonalise_case("hidden 2048x2048", 1, 2048, 2048, "float32"),
        # the largest: an odd-sided wide matrix of a large layer
        orthogonalise_case("wide 4095x6001", 1, 4095, 6001, "bfloat16"),
        # one optimiser step over the matrices of a four-layer network (kernel weights and head)
        muon_case("network of four layers", "8x5,16x40,32x80,64x160,128x64,40x128", "float32"),
        # one optimiser step over the matrices of a transformer-sized block: square, wide and tall, ragged
        muon_case("block of large matrices", "1024x1024,1024x1024,1024x2730,2730x1024", "float32"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["log_probabilities", "log_probabilities", "orthogonalise", "orthogonalise", "muon"])
    if op == "log_probabilities":
        classes = _log_int(rng, 2, 131072)
        rows = _log_int(rng, 1, max(1, min(8192, 100_000_000 // classes)))
        n_top = min(classes, rng.choice([0, 0, 1, 3, 5, 8, 20, 32]))
        case = log_probs_case("", rows, classes, rng.choice(["float32", "bfloat16", "float16"]), n_top, rng.random() < 0.5,
                              rng.choice([1.0, 0.7, 1.5]), rng.choice([0.0, 0.0, 0.02, 0.3]))
    elif op == "orthogonalise":
        rows, cols = _log_int(rng, 1, 3000), _log_int(rng, 1, 6000)
        batch = _log_int(rng, 1, max(1, min(48, 12_000_000 // (rows * cols))))
        case = orthogonalise_case("", batch, rows, cols, rng.choice(["float32", "bfloat16"]))
    else:
        top = rng.choice([160, 700, 2000])
        shapes = ",".join(f"{_log_int(rng, 2, top)}x{_log_int(rng, 2, top)}" for _ in range(rng.randint(1, 8)))
        case = muon_case("", shapes, rng.choice(["float32", "bfloat16"]), rng.random() < 0.7)
    del case["name"]
    return case


def _shapes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["shapes"].split(",")]


def _updates(g, batch, rows, cols):
    """What gradients of weight matrices look like: a few strong directions over a floor of noise."""
    rank = max(1, min(rows, cols, 24) // 2)
    left = torch.randn(batch, rows, rank, generator=g, device="cuda")
    right = torch.randn(batch, rank, cols, generator=g, device="cuda")
    strength = torch.exp(-0.35 * torch.arange(rank, device="cuda"))
    noise = torch.randn(batch, rows, cols, generator=g, device="cuda")
    return 1e-3 * ((left * strength) @ right + 0.2 * noise)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 11)
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "log_probabilities":
        n, c = case["rows"], case["classes"]
        logits = torch.randn(n, c, generator=g, device="cuda")
        # likelier and rarer classes, the way a vocabulary has them
        logits = 2.0 * logits - 1.2 * torch.log(1.0 + torch.randperm(c, generator=g, device="cuda").float())
        targets = torch.randint(0, c, (n,), generator=g, device="cuda")
        likely = (logits + torch.randn(n, c, generator=g, device="cuda")).argmax(dim=1)
        targets = torch.where(torch.rand(n, generator=g, device="cuda") < 0.8, likely, targets)
        n_masked = min(c - 1, int(case["masked"] * c))
        if n_masked:
            # padding entries of the vocabulary; no target is one of them
            logits[:, c - n_masked:] = -math.inf
            targets = torch.where(targets >= c - n_masked, targets % (c - n_masked), targets)
        if n > 4:
            targets = torch.where(torch.rand(n, generator=g, device="cuda") < 0.1, IGNORED, targets)
        state = {"case": case, "logits": logits.to(dtype), "targets": targets}
        if case["train"]:
            state["grad_target"] = torch.randn(n, generator=g, device="cuda")
            state["grad_entropy"] = 0.1 * torch.randn(n, generator=g, device="cuda")
            state["grad_top"] = 0.3 * torch.randn(n, case["n_top"], generator=g, device="cuda")
        return state
    if case["op"] == "orthogonalise":
        return {"case": case, "update": _updates(g, case["batch"], case["rows"], case["cols"]).to(dtype)}
    shapes = _shapes(case)
    return {"case": case,
            "params": [(torch.randn(m, n, generator=g, device="cuda") / math.sqrt(n)).to(dtype) for m, n in shapes],
            "grads": [_updates(g, 1, m, n)[0].to(dtype) for m, n in shapes],
            "momenta": [0.7 * _updates(g, 1, m, n)[0] for m, n in shapes]}


LR, MOMENTUM, WEIGHT_DECAY = 0.02, 0.95, 0.01


# ---- plain forms -----------------------------------------------------------------------------------------------------

def _top_plain(x, n_top):
    """The n_top largest of each row, ties to the lowest index: one 64-bit key of (order of the value, index)."""
    bits = torch.where(x == 0, 0.0, x).view(torch.int32)
    order = torch.where(bits >= 0, bits, bits ^ 0x7FFFFFFF).long()
    index = torch.arange(x.shape[1], device=x.device)
    return 0x7FFFFFFF - (((order << 32) | (0x7FFFFFFF - index)).topk(n_top, dim=1).values & 0xFFFFFFFF)


def _log_probabilities_plain(s):
    case, targets = s["case"], s["targets"]
    z = s["logits"].float()
    x = z if case["temperature"] == 1.0 else z / case["temperature"]
    x = x - x.amax(dim=1, keepdim=True)
    e = torch.exp(x)
    total = e.sum(dim=1, keepdim=True)
    log_p = x - torch.log(total)
    p = e / total
    entropy = -torch.where(p > 0, p * log_p, 0.0).sum(dim=1)
    kept = targets != IGNORED
    at = torch.where(kept, targets, 0).unsqueeze(1)
    out = [torch.where(kept, log_p.gather(1, at).squeeze(1), 0.0), entropy]
    if case["n_top"]:
        top = _top_plain(z, case["n_top"])
        out += [log_p.gather(1, top), top]
    if case["train"]:
        g_target = torch.where(kept, s["grad_target"], 0.0).unsqueeze(1)
        g_sum = g_target + s["grad_top"].sum(dim=1, keepdim=True)
        g_entropy = s["grad_entropy"].unsqueeze(1)
        grad = -p * g_sum - torch.where(p > 0, p * g_entropy * (log_p + entropy.unsqueeze(1)), 0.0)
        grad = grad.scatter_add(1, at, g_target)
        if case["n_top"]:
            grad = grad.scatter_add(1, top, s["grad_top"])
        out.append((grad / case["temperature"]).to(s["logits"].dtype))
    return out


def _newton_schulz_plain(update):
    """update [..., m, n] in 32 bits -> the Newton-Schulz iterate of update / |update|."""
    x = update.transpose(-1, -2) if update.shape[-2] > update.shape[-1] else update
    x = x / (x.square().sum(dim=(-1, -2), keepdim=True).sqrt() + EPSILON)
    a, b, c = COEFFICIENTS
    for _ in range(STEPS):
        gram = x @ x.transpose(-1, -2)
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.transpose(-1, -2) if update.shape[-2] > update.shape[-1] else x


def _muon_plain(s):
    for p, g, m in zip(s["params"], s["grads"], s["momenta"]):
        g = g.float()
        m.mul_(MOMENTUM).add_(g, alpha=1 - MOMENTUM)
        update = (1 - MOMENTUM) * g + MOMENTUM * m if s["case"]["nesterov"] else m
        scale = LR * math.sqrt(max(1.0, p.shape[0] / p.shape[1]))
        p.copy_(p.float() * (1 - LR * WEIGHT_DECAY) - scale * _newton_schulz_plain(update))
    return [s["params"], s["momenta"]]


# ---- the framework's calls -------------------------------------------------------------------------------------------

def _run_own(s):
    if PACKAGE not in sys.path:
        sys.path.insert(0, PACKAGE)
    import gmc.classification
    import gmc.optimisation
    case = s["case"]
    if case["op"] == "orthogonalise":
        return gmc.optimisation.orthogonalise(s["update"], steps=STEPS, coefficients=COEFFICIENTS, epsilon=EPSILON)
    if case["op"] == "muon":
        gmc.optimisation.muon_update(s["params"], s["grads"], s["momenta"], lr=LR, momentum=MOMENTUM,
                                     weight_decay=WEIGHT_DECAY, nesterov=case["nesterov"], steps=STEPS,
                                     coefficients=COEFFICIENTS, epsilon=EPSILON)
        return [s["params"], s["momenta"]]
    logits = s["logits"].detach().requires_grad_(True) if case["train"] else s["logits"]
    r = gmc.classification.log_probabilities(logits, s["targets"], n_top=case["n_top"], temperature=case["temperature"],
                                             ignore_index=IGNORED)
    out = [r.target, r.entropy]
    if case["n_top"]:
        out += [r.top, r.top_indices]
    if case["train"]:
        values, grads = [r.target, r.entropy], [s["grad_target"], s["grad_entropy"]]
        if case["n_top"]:
            values, grads = values + [r.top], grads + [s["grad_top"]]
        out.append(torch.autograd.grad(values, logits, grads)[0])
    return out


def run(state):
    if own:
        return _run_own(state)
    if state["case"]["op"] == "log_probabilities":
        return _log_probabilities_plain(state)
    if state["case"]["op"] == "orthogonalise":
        return _newton_schulz_plain(state["update"].float()).to(state["update"].dtype)
    return _muon_plain(state)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------

def _newton_schulz_flops(m, n):
    """Two products with a symmetric result (half of their sums are needed) and one general product per step."""
    m, n = min(m, n), max(m, n)
    return STEPS * (m * (m + 1) * n + m * (m + 1) * m + 2 * m * m * n)


def work(case):
    size = DTYPES[case["dtype"]].itemsize
    if case["op"] == "log_probabilities":
        n, c, k = case["rows"], case["classes"], case["n_top"]
        if case["train"]:
            return {"bytes": 2 * n * c * size + n * (8 + 8 + 8) + n * k * (4 + 8 + 4), "flops": 12 * n * c}
        return {"bytes": n * c * size + n * (8 + 8) + n * k * (4 + 8), "flops": 6 * n * c}
    if case["op"] == "orthogonalise":
        b, m, n = case["batch"], case["rows"], case["cols"]
        return {"bytes": 2 * b * m * n * size, "flops": b * _newton_schulz_flops(m, n)}
    shapes = _shapes(case)
    return {"bytes": sum(m * n * (3 * size + 8) for m, n in shapes),
            "flops": sum(_newton_schulz_flops(m, n) + 9 * m * n for m, n in shapes)}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------

def _log_probabilities_exact(s):
    """Row blocks; the gradient as the vector-Jacobian product of 64-bit log-probabilities by automatic differentiation."""
    case, blocks = s["case"], []
    step = max(1, 16_000_000 // case["classes"])
    for at in range(0, case["rows"], step):
        rows = slice(at, at + step)
        z = s["logits"][rows].double().requires_grad_(case["train"])
        log_p = torch.log_softmax(z / case["temperature"], dim=1)
        finite = torch.where(torch.isinf(log_p), 0.0, log_p)
        entropy = -(log_p.exp() * finite).sum(dim=1)
        targets = s["targets"][rows]
        picked = log_p.gather(1, targets.clamp_min(0).unsqueeze(1)).squeeze(1)
        target = torch.where(targets == IGNORED, torch.zeros_like(picked), picked)
        out = [target.detach(), entropy.detach()]
        values = (target * s["grad_target"][rows]).sum() + (entropy * s["grad_entropy"][rows]).sum() if case["train"] else None
        if case["n_top"]:
            index = torch.sort(z.detach(), dim=1, descending=True, stable=True).indices[:, :case["n_top"]]
            top = log_p.gather(1, index)
            out += [top.detach(), index]
            if case["train"]:
                values = values + (top * s["grad_top"][rows]).sum()
        if case["train"]:
            out.append(torch.autograd.grad(values, z)[0])
        blocks.append(out)
    return [torch.cat(parts) for parts in zip(*blocks)]


def _newton_schulz_exact(update):
    """The iterate is f(XX^T) X with a polynomial f: taken on the eigenvalues of XX^T instead of by products."""
    x = update.double()
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    x = x / (torch.linalg.matrix_norm(x, keepdim=True) + EPSILON)
    lam, vec = torch.linalg.eigh(x @ x.mT)
    f = torch.ones_like(lam)
    for _ in range(STEPS):
        now = lam * f * f
        f = f * (COEFFICIENTS[0] + now * (COEFFICIENTS[1] + COEFFICIENTS[2] * now))
    x = (vec * f.unsqueeze(-2)) @ (vec.mT @ x)
    return x.mT if tall else x


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "log_probabilities":
        return _log_probabilities_exact(s)
    if case["op"] == "orthogonalise":
        return _newton_schulz_exact(s["update"])
    params, momenta = [], []
    for p, g, m in zip(s["params"], s["grads"], s["momenta"]):
        m = MOMENTUM * m.double() + (1 - MOMENTUM) * g.double()
        update = m + (1 - MOMENTUM) * (g.double() - m) if case["nesterov"] else m
        scale = LR * math.sqrt(max(1.0, p.shape[0] / p.shape[1]))
        params.append((1 - LR * WEIGHT_DECAY) * p.double() - scale * _newton_schulz_exact(update))
        momenta.append(m)
    return [params, momenta]
