"""Cases and plain forms of the operators of a training step that ends in many classes: the loss of a linear head over a
large set of classes without its logits, with its gradients (`linear_cross_entropy`), the orthogonalised update of weight
matrices (`muon_step`), and the Newton-Schulz orthogonalisation by itself (`newton_schulz`).

`own` false: elementary torch operations in fp32.  `own` true: the calls of origindl_b200.ops.
"""
import math

import torch

own = False

NS_A, NS_B, NS_C = 3.4445, -4.7750, 2.0315
EPS = 1e-7
IGNORE = -100

# the range the listed cases stand for (draw() keeps every case's products below the largest listed case's)
MOST_LCE = 6 * 8192 * 131072 * 2048
MOST_NS = 5 * 4 * 8192**3


def listed():
    return [
        # the head of the small image classifier, one step at its batch: latency
        dict(name="lce_classifier_head", op="lce", rows=512, classes=10, features=1000, layout="in_out", bias=True,
             grad=True, ignored=0.0, labels="int32"),
        # the head of the deep wide MLP at its batch
        dict(name="lce_wide_mlp_head", op="lce", rows=8192, classes=1000, features=4096, layout="in_out", bias=True,
             grad=True, ignored=0.0, labels="int32"),
        # scoring one position against a vocabulary: one read of the weights
        dict(name="lce_score_one", op="lce", rows=1, classes=32000, features=2048, layout="out_in", bias=False,
             grad=False, ignored=0.0, labels="int64"),
        # scoring a few short candidates
        dict(name="lce_score_few", op="lce", rows=40, classes=50021, features=1024, layout="out_in", bias=False,
             grad=False, ignored=0.1, labels="int64"),
        # a padded batch, nothing of whose sizes divides anything
        dict(name="lce_ragged_batch", op="lce", rows=1999, classes=50021, features=1001, layout="out_in", bias=True,
             grad=True, ignored=0.2, labels="int64"),
        # evaluation of a long batch: the loss alone
        dict(name="lce_evaluate", op="lce", rows=4096, classes=65536, features=1024, layout="out_in", bias=False,
             grad=False, ignored=0.05, labels="int64"),
        # a full training batch over a large vocabulary
        dict(name="lce_train_large", op="lce", rows=8192, classes=131072, features=2048, layout="out_in", bias=False,
             grad=True, ignored=0.02, labels="int64"),
        # first layer of the small image classifier: latency
        dict(name="muon_classifier", op="muon", batch=1, rows=784, cols=1000, layout="in_out", nesterov=True, decay=1e-4),
        # the equal-shaped projections of a stack of layers in one call
        dict(name="muon_stack", op="muon", batch=12, rows=1024, cols=1024, layout="out_in", nesterov=True, decay=0.1),
        # one hidden layer of the widest MLP
        dict(name="muon_wide_mlp", op="muon", batch=1, rows=8192, cols=8192, layout="in_out", nesterov=True, decay=0.0),
        # a tall odd matrix, orthogonalised by itself
        dict(name="ns_tall_odd", op="ns", batch=1, rows=4099, cols=1023),
        # wide ones: several small heads at once
        dict(name="ns_small_heads", op="ns", batch=32, rows=64, cols=512),
    ]


def _size(rng, low, high):
    """Log-uniform between low and high; two in five are rounded to a multiple of 64, the rest stay as they fall."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return max(low, min(high, v // 64 * 64)) if v >= 128 and rng.random() < 0.4 else v


def draw(rng):
    if rng.random() < 0.55:
        while True:
            c = dict(op="lce", rows=_size(rng, 1, 8192), classes=_size(rng, 2, 131072), features=_size(rng, 16, 4096),
                     layout=rng.choice(["in_out", "out_in"]), bias=rng.random() < 0.5, grad=rng.random() < 0.6,
                     ignored=rng.choice([0.0, 0.05, 0.5]), labels=rng.choice(["int32", "int64"]))
            if 6 * c["rows"] * c["classes"] * c["features"] <= MOST_LCE:
                return c
    while True:
        op = rng.choice(["muon", "muon", "ns"])
        c = dict(op=op, batch=_size(rng, 1, 24), rows=_size(rng, 4, 8192), cols=_size(rng, 4, 8192))
        s, m = sorted((c["rows"], c["cols"]))
        if c["batch"] * s * m <= 8192**2 and 5 * c["batch"] * (s**3 + 3 * s * s * m) <= MOST_NS:
            if op == "muon":
                c.update(layout=rng.choice(["in_out", "out_in"]), nesterov=rng.random() < 0.7,
                         decay=rng.choice([0.0, 1e-4, 0.1]))
            return c


def _normal(gen, *shape, scale=1.0):
    return torch.randn(*shape, device="cuda", generator=gen).mul_(scale)


def _gradient(gen, batch, rows, cols):
    """A weight gradient: a few strong directions of decaying size on a floor of noise."""
    rank = max(1, min(rows, cols) // 16)
    size = torch.arange(1, rank + 1, device="cuda", dtype=torch.float32).rsqrt()
    g = (_normal(gen, batch, rows, rank) * size) @ _normal(gen, batch, rank, cols)
    return g.mul_(1e-3).add_(_normal(gen, batch, rows, cols), alpha=3e-4)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    c = case
    if c["op"] == "lce":
        m, n, k = c["rows"], c["classes"], c["features"]
        w = _normal(gen, n, k, scale=0.7 / math.sqrt(k))
        # frequent classes are drawn more often, and the features lean towards their class: some rows are already sure
        u = torch.rand(m, device="cuda", generator=gen, dtype=torch.float64)
        labels = (n ** u - 1).long().clamp_(0, n - 1)
        lean = torch.rand(m, 1, device="cuda", generator=gen) * 12
        x = _normal(gen, m, k) + lean * w[labels]
        if c["ignored"]:
            labels[torch.rand(m, device="cuda", generator=gen) < c["ignored"]] = IGNORE
        if c["layout"] == "in_out":
            w = w.t().contiguous()
        b = _normal(gen, n, scale=0.1) if c["bias"] else None
        labels = labels.to(torch.int32 if c["labels"] == "int32" else torch.int64)
        return dict(case=dict(c), x=x, w=w, b=b, labels=labels)
    grad = _gradient(gen, c["batch"], c["rows"], c["cols"])
    if c["op"] == "ns":
        return dict(case=dict(c), grad=grad)
    param = _normal(gen, c["batch"], c["rows"], c["cols"], scale=0.02)
    buf = _gradient(gen, c["batch"], c["rows"], c["cols"]).mul_(5).add_(grad, alpha=10)
    return dict(case=dict(c), grad=grad, param=param, buf=buf)


def _plain_lce(x, w, b, labels, in_out, need_grad):
    logits = x @ w if in_out else x @ w.t()
    if b is not None:
        logits += b
    top = logits.max(dim=1, keepdim=True).values
    lse = top + torch.log(torch.exp(logits - top).sum(dim=1, keepdim=True))
    valid = labels != IGNORE
    count = valid.sum().clamp(min=1)
    at = torch.where(valid, labels, torch.zeros_like(labels)).long()[:, None]
    picked = logits.gather(1, at)
    loss = torch.where(valid, (lse - picked)[:, 0], torch.zeros_like(lse[:, 0])).sum() / count
    # a row without a label is not evaluated: its log-sum-exp is given as 0
    out = dict(loss=loss, lse=torch.where(valid, lse[:, 0], torch.zeros_like(lse[:, 0])))
    if not need_grad:
        return out
    d = logits.sub_(lse).exp_()
    d.scatter_add_(1, at, torch.full_like(lse, -1.0))
    d *= torch.where(valid, 1.0 / count, torch.zeros((), device=x.device))[:, None]
    out["dx"] = d @ w.t() if in_out else d @ w
    out["dw"] = x.t() @ d if in_out else d.t() @ x
    if b is not None:
        out["db"] = d.sum(dim=0)
    return out


def _plain_ns(g, steps=5):
    tall = g.shape[-2] > g.shape[-1]
    x = g.transpose(-1, -2) if tall else g
    norm = x.double().square().sum(dim=(-1, -2), keepdim=True).sqrt().clamp(min=EPS)
    x = (x / norm).float()
    for _ in range(steps):
        a = x @ x.transpose(-1, -2)
        x = NS_A * x + (NS_B * a + NS_C * (a @ a)) @ x
    return x.transpose(-1, -2).contiguous() if tall else x


def _lr_factor(c):
    fan_out, fan_in = (c["rows"], c["cols"]) if c["layout"] == "out_in" else (c["cols"], c["rows"])
    return math.sqrt(max(1.0, fan_out / fan_in))


LR, MOMENTUM = 0.02, 0.95


def _plain_muon(s):
    c = s["case"]
    s["buf"].mul_(MOMENTUM).add_(s["grad"])
    u = s["grad"] + MOMENTUM * s["buf"] if c["nesterov"] else s["buf"]
    u = _plain_ns(u)
    s["param"].mul_(1 - LR * c["decay"]).sub_(u, alpha=LR * _lr_factor(c))
    return dict(param=s["param"], buf=s["buf"])


def run(state):
    c = state["case"]
    if own:
        from origindl_b200 import capi, ops

        capi.init(0)
        if c["op"] == "lce":
            loss, lse, dx, dw, db = ops.linear_cross_entropy(
                state["x"], state["w"], state["labels"], b=state["b"], ignore_index=IGNORE,
                w_layout=ops.W_IN_OUT if c["layout"] == "in_out" else ops.W_OUT_IN, need_dx=c["grad"], need_dw=c["grad"],
                need_db=c["grad"] and c["bias"])
            out = dict(loss=loss, lse=lse, dx=dx, dw=dw, db=db)
            return {k: v for k, v in out.items() if v is not None}
        if c["op"] == "ns":
            return dict(out=ops.newton_schulz(state["grad"], steps=5, eps=EPS))
        ops.muon_step(state["param"], state["grad"], state["buf"], lr=LR, momentum=MOMENTUM, nesterov=c["nesterov"],
                      weight_decay=c["decay"], steps=5, eps=EPS,
                      w_layout=ops.W_IN_OUT if c["layout"] == "in_out" else ops.W_OUT_IN)
        return dict(param=state["param"], buf=state["buf"])
    if c["op"] == "lce":
        return _plain_lce(state["x"], state["w"], state["b"], state["labels"], c["layout"] == "in_out", c["grad"])
    if c["op"] == "ns":
        return dict(out=_plain_ns(state["grad"]))
    return _plain_muon(state)


def work(case):
    c = case
    if c["op"] == "lce":
        m, n, k = c["rows"], c["classes"], c["features"]
        nbytes = 4 * (m * k + n * k + m + 1) + m * (4 if c["labels"] == "int32" else 8) + (4 * n if c["bias"] else 0)
        if c["grad"]:
            nbytes += 4 * (m * k + n * k) + (4 * n if c["bias"] else 0)
        return {"bytes": nbytes, "flops": (6 if c["grad"] else 2) * m * n * k}
    s, l = sorted((c["rows"], c["cols"]))
    # X X^T and A^2 are symmetric: half of each is enough
    flops = c["batch"] * 5 * (s * s * l + s**3 + 2 * s * s * l)
    return {"bytes": c["batch"] * s * l * (20 if c["op"] == "muon" else 8), "flops": flops}


# ---- the definitions in 64 bits, apart from the plain forms --------------------------------------------------------------
def _exact_lce(s):
    c = s["case"]
    x, labels = s["x"].double(), s["labels"].long()
    w = s["w"].double() if c["layout"] == "out_in" else s["w"].double().t()
    z = torch.einsum("mk,nk->mn", x, w)
    if s["b"] is not None:
        z = z + s["b"].double()
    lse = torch.logsumexp(z, dim=1)
    rows = torch.nonzero(labels != IGNORE)[:, 0]
    n_valid = max(1, rows.numel())
    loss = (lse[rows] - z[rows, labels[rows]]).sum() / n_valid
    out = dict(loss=loss, lse=torch.zeros_like(lse).index_copy(0, rows, lse[rows]))
    if c["grad"]:
        p = torch.zeros_like(z)
        p[rows] = torch.exp(z[rows] - lse[rows, None]) / n_valid
        del z
        p[rows, labels[rows]] -= 1.0 / n_valid
        out["dx"] = torch.einsum("mn,nk->mk", p, w)
        dw = torch.einsum("mn,mk->nk", p, x)
        out["dw"] = dw if c["layout"] == "out_in" else dw.t().contiguous()
        if s["b"] is not None:
            out["db"] = p.sum(0)
    return out


def _exact_ns(g):
    x = g / torch.linalg.matrix_norm(g, keepdim=True).clamp(min=EPS)
    for _ in range(5):
        if x.shape[-2] <= x.shape[-1]:
            gram = x @ x.mT
            x = NS_A * x + NS_B * (gram @ x) + NS_C * (gram @ (gram @ x))
        else:
            gram = x.mT @ x
            x = NS_A * x + NS_B * (x @ gram) + NS_C * ((x @ gram) @ gram)
    return x


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["op"] == "lce":
        return _exact_lce(s)
    g = s["grad"].double()
    if c["op"] == "ns":
        return dict(out=_exact_ns(g))
    buf = MOMENTUM * s["buf"].double() + g
    u = _exact_ns(g + MOMENTUM * buf if c["nesterov"] else buf)
    param = s["param"].double() * (1 - LR * c["decay"]) - LR * _lr_factor(c) * u
    return dict(param=param, buf=buf)
