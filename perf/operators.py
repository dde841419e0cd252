"""Cases for the operators around a decoder's matrices: the token table and its gradient, the RMS norm of the residual stream
and its adjoint, and the Muon update of the weight matrices.

`run` computes a case either in its plain form (elementary torch operations, 32 bits, rounded once at the end) or, with `own`
set, as the programs of this package on the same tensors, which `prepare` has imported as pool buffers.  `exact` restates every
operator in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ITEM = {"f32": 4, "bf16": 2, "f16": 2}
NS = (3.4445, -4.7750, 2.0315)      # the quintic whose five steps bring singular values near 1
STEPS, NORM_EPS = 5, 1e-7
E4M3_MAX, AMAX_FLOOR = 448.0, 1e-30
RMS_EPS = 1e-6


def listed():
    return [
        # the table read for one decoding step of a small batch: launch latency
        dict(name="embed step bf16", op="embed", dtype="bf16", tokens=8, vocab=32000, dim=2048, pad=0.0, scale=1.0),
        # the table read of one training batch, eight sequences of 2048 tokens
        dict(name="embed batch bf16", op="embed", dtype="bf16", tokens=16384, vocab=50257, dim=2048, pad=0.0, scale=45.25),
        # its gradient: a few words make up much of the text, most of the table is not met
        dict(name="embed grad bf16", op="embed_bwd", dtype="bf16", tokens=16384, vocab=50257, dim=2048, pad=0.0, scale=45.25, accumulate=False),
        # a small table with an odd width, padded sequences, added to the gradient that a tied output layer has left there
        dict(name="embed grad f32 add", op="embed_bwd", dtype="f32", tokens=4099, vocab=1021, dim=777, pad=0.25, scale=1.0, accumulate=True),
        # the norm of one decoding step of a small batch
        dict(name="rms step bf16", op="rms", dtype="bf16", rows=4, cols=4096, residual=True, quant=False, group=0),
        # the norm in front of a training step's projections, with the residual stream written beside it
        dict(name="rms block bf16", op="rms", dtype="bf16", rows=16384, cols=2048, residual=True, quant=False, group=0),
        # the same in front of a product that reads 8 bits with a scale for each 128 columns
        dict(name="rms e4m3 bf16", op="rms", dtype="bf16", rows=8192, cols=4096, residual=True, quant=True, group=128),
        # the adjoint in a training step: input gradient with the residual stream's own added, and the weight's
        dict(name="rms grad bf16", op="rms_bwd", dtype="bf16", rows=16384, cols=2048, residual=True),
        # the same in full precision at an odd width
        dict(name="rms grad f32", op="rms_bwd", dtype="f32", rows=1000, cols=5003, residual=False),
        # one layer of a small classifier
        dict(name="muon small f32", op="muon", dtype="f32", count=1, rows=128, cols=784),
        # the four projections of a transformer block, updated together
        dict(name="muon block bf16", op="muon", dtype="bf16", count=4, rows=2048, cols=2048),
        # a feed-forward layer's expanding matrix in full precision
        dict(name="muon ffn f32", op="muon", dtype="f32", count=1, rows=8192, cols=2048),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["embed", "embed_bwd", "rms", "rms_bwd", "muon"])
    dtype = rng.choice(["bf16", "f16", "f32"])
    if op in ("embed", "embed_bwd"):
        c = dict(op=op, dtype=dtype, tokens=_log(rng, 1, 32768), vocab=_log(rng, 256, 65536), dim=_log(rng, 64, 4096),
                 pad=rng.choice([0.0, 0.1, 0.4]), scale=rng.choice([1.0, 8.0, 22.6]))
        if op == "embed_bwd":
            c["accumulate"] = rng.random() < 0.3
        return c
    if op == "muon":
        c = dict(op=op, dtype=dtype, count=rng.randint(1, 4), rows=_log(rng, 32, 4096), cols=_log(rng, 32, 4096))
        while work(c)["flops"] > 6e11:      # no more than the largest listed update
            c["count"], c["rows"] = max(1, c["count"] - 1), c["rows"] if c["count"] > 1 else c["rows"] * 3 // 4
        return c
    c = dict(op=op, dtype=dtype, rows=_log(rng, 1, 16384), cols=_log(rng, 64, 8192), residual=rng.random() < 0.7)
    if op == "rms":
        c["quant"] = rng.random() < 0.4
        c["group"] = rng.choice([0, 64, 128]) if c["quant"] else 0
    return c


# ---- inputs ---------------------------------------------------------------------------------------------------------------
def _ids(case, gen):
    """Token numbers as text has them: the frequency of a word falls with its rank, the ranks lie scattered over the table; the
    given share of positions is padding (-1) at the end of the sequence."""
    n, vocab = case["tokens"], case["vocab"]
    u = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64)
    rank = (torch.pow(torch.tensor(float(vocab), device="cuda", dtype=torch.float64), u) - 1.0).long().clamp(0, vocab - 1)
    ids = torch.randperm(vocab, generator=gen, device="cuda")[rank].to(torch.int32)
    used = n - int(n * case["pad"])
    ids[used:] = -1
    return ids


def _inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    t = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0):
        return torch.randn(*shape, generator=gen, device="cuda").mul_(std).add_(mean).to(t)

    op = case["op"]
    if op == "embed":
        return dict(ids=_ids(case, gen), table=normal(case["vocab"], case["dim"], std=0.02))
    if op == "embed_bwd":
        s = dict(ids=_ids(case, gen), dout=normal(case["tokens"], case["dim"], std=0.1))
        s["dtable"] = normal(case["vocab"], case["dim"], std=0.1) if case["accumulate"] else torch.zeros(case["vocab"], case["dim"], device="cuda", dtype=t)
        return s
    if op == "rms":
        s = dict(x=normal(case["rows"], case["cols"]), weight=normal(case["cols"], std=0.2, mean=1.0))
        if case["residual"]:
            s["residual"] = normal(case["rows"], case["cols"], std=2.0)
        return s
    if op == "rms_bwd":
        s = dict(h=normal(case["rows"], case["cols"], std=2.0), dy=normal(case["rows"], case["cols"], std=0.1),
                 weight=normal(case["cols"], std=0.2, mean=1.0))
        if case["residual"]:
            s["dh"] = normal(case["rows"], case["cols"], std=0.1)
        return s
    # a gradient of a few strong directions over a broad floor, as a layer's is
    n, r, c = case["count"], case["rows"], case["cols"]
    k = max(1, min(r, c) // 16)
    strong = torch.randn(n, r, k, generator=gen, device="cuda") @ torch.randn(n, k, c, generator=gen, device="cuda")
    grads = (strong.div_(math.sqrt(k)).add_(torch.randn(n, r, c, generator=gen, device="cuda"))).mul_(1e-3).to(t)
    return dict(p=[normal(r, c, std=0.02) for _ in range(n)], g=[grads[i].clone() for i in range(n)], buf=[normal(r, c, std=1e-3) for _ in range(n)])


MUON = dict(lr=0.02, weight_decay=0.01, momentum=0.95)


class _Program:
    """A program of the package on tensors of this process: they are imported as pool buffers, in the order of its arguments, and the
    launches go to torch's stream, in order with what fills the tensors before and reads or frees them after."""

    def __init__(self, desc, tensors):
        from zyx_b200.ops import Session
        if not hasattr(_Program, "session"):
            _Program.session = Session(device_ids=[torch.cuda.current_device()], round_nearest=True)
        s = _Program.session
        self.pool, self.device = s.pool, s.device
        self.device.use_stream(torch.cuda.current_stream().cuda_stream)
        self.prog = self.device.create_program(desc)
        self.args = [self.pool.import_device(x.data_ptr(), x.numel() * x.element_size()) for x in tensors]

    def __call__(self):
        self.device.launch(self.prog, self.args)

    def __del__(self):
        try:
            for b in self.args:
                self.pool.deallocate(b)
            self.device.release(self.prog)
        except Exception:       # an interpreter that is ending
            pass


def _program(case, s):
    """What a user of the package keeps for this path: the outputs' memory and the program."""
    from zyx_b200 import _lib as L
    from zyx_b200 import backend as B
    dt = {"f32": L.F32, "bf16": L.BF16, "f16": L.F16}[case["dtype"]]
    op = case["op"]
    if op == "embed":
        s["out"] = torch.empty(case["tokens"], case["dim"], device="cuda", dtype=s["table"].dtype)
        return _Program(B.embedding_desc(dt, case["tokens"], case["vocab"], case["dim"], scale=case["scale"]), [s["ids"], s["table"], s["out"]])
    if op == "embed_bwd":
        d = B.embedding_desc(dt, case["tokens"], case["vocab"], case["dim"], scale=case["scale"], backward=True, accumulate=case["accumulate"])
        return _Program(d, [s["ids"], s["dout"], s["dtable"]])
    if op == "rms":
        rows, cols = case["rows"], case["cols"]
        d = B.rmsnorm_desc(dt, rows, cols, eps=RMS_EPS, has_residual=case["residual"], has_weight=True, quant=case["quant"], group=case["group"])
        args = [s["x"]] + ([s["residual"]] if case["residual"] else []) + [s["weight"]]
        if case["residual"]:
            s["h"] = torch.empty_like(s["x"])
            args.append(s["h"])
        if case["quant"]:
            s["y"] = torch.empty(rows, cols, device="cuda", dtype=torch.float8_e4m3fn)
            s["scales"] = torch.empty(rows, -(-cols // (case["group"] or cols)), device="cuda")
            args += [s["y"], s["scales"]]
        else:
            s["y"] = torch.empty_like(s["x"])
            args.append(s["y"])
        return _Program(d, args)
    if op == "rms_bwd":
        d = B.rmsnorm_desc(dt, case["rows"], case["cols"], eps=RMS_EPS, has_weight=True, backward=True, has_dh=case["residual"])
        s["dx"], s["dweight"] = torch.empty_like(s["h"]), torch.empty_like(s["weight"])
        return _Program(d, [s["h"], s["dy"], s["weight"]] + ([s["dh"]] if case["residual"] else []) + [s["dx"], s["dweight"]])
    d = B.muon_desc(dt, [(case["rows"], case["cols"])] * case["count"], nesterov=True, steps=STEPS, coefficients=NS, eps=NORM_EPS, **MUON)
    return _Program(d, s["p"] + s["g"] + s["buf"])


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        s["program"] = _program(case, s)
    return s


# ---- plain forms ------------------------------------------------------------------------------------------------------------
def _embed(s, case):
    ids, vocab = s["ids"], case["vocab"]
    met = (ids >= 0) & (ids < vocab)
    rows = s["table"][ids.clamp(0, vocab - 1).long()].float() * case["scale"]
    return dict(out=torch.where(met[:, None], rows, 0.0).to(s["table"].dtype))


def _embed_bwd(s, case):
    ids, vocab, d = s["ids"], case["vocab"], s["dtable"]
    met = (ids >= 0) & (ids < vocab)
    rows = torch.where(met[:, None], s["dout"].float(), 0.0)
    total = torch.zeros(vocab, case["dim"], device="cuda").index_add_(0, ids.clamp(0, vocab - 1).long(), rows) * case["scale"]
    d.copy_(d.float() + total if case["accumulate"] else total)
    return dict(dtable=d)


def _groups(y, group):
    """[rows, cols] as [rows, groups, group], zeros behind the last column."""
    rows, cols = y.shape
    n = -(-cols // group)
    return torch.nn.functional.pad(y, (0, n * group - cols)).view(rows, n, group)


def _rms(s, case):
    x = s["x"]
    out = {}
    h = x.float()
    if case["residual"]:
        h = h + s["residual"].float()
        out["h"] = h.to(x.dtype)
    y = h * torch.rsqrt((h * h).mean(1, keepdim=True) + RMS_EPS) * s["weight"].float()
    if not case["quant"]:
        out["y"] = y.to(x.dtype)
        return out
    g = _groups(y, case["group"] or case["cols"])
    scales = g.abs().amax(2).clamp_min(AMAX_FLOOR) / E4M3_MAX
    q = (g / scales[:, :, None]).clamp(-E4M3_MAX, E4M3_MAX).reshape(case["rows"], -1)[:, :case["cols"]]
    return dict(out, y=q.to(torch.float8_e4m3fn).contiguous(), scales=scales)


def _rms_bwd(s, case):
    h, dy, w = s["h"].float(), s["dy"].float(), s["weight"].float()
    rstd = torch.rsqrt((h * h).mean(1, keepdim=True) + RMS_EPS)
    xhat = h * rstd
    g = dy * w
    dx = rstd * (g - xhat * (g * xhat).mean(1, keepdim=True))
    if case["residual"]:
        dx = dx + s["dh"].float()
    return dict(dx=dx.to(s["h"].dtype), dweight=(dy * xhat).sum(0).to(s["weight"].dtype))


def _adjust(case):
    return math.sqrt(max(1.0, case["rows"] / case["cols"]))


def _muon(s, case):
    t = s["p"][0].dtype
    g, buf, p = torch.stack(s["g"]).float(), torch.stack(s["buf"]).float(), torch.stack(s["p"]).float()
    buf = (buf * MUON["momentum"] + g).to(t)
    u = g + MUON["momentum"] * buf.float()
    norm = u.double().square().sum((1, 2), keepdim=True).sqrt().float()
    x = u / (norm + NORM_EPS)
    tall = case["rows"] > case["cols"]
    x = x.transpose(1, 2) if tall else x
    for _ in range(STEPS):
        a = x @ x.transpose(1, 2)
        x = NS[0] * x + (NS[1] * a + NS[2] * (a @ a)) @ x
    x = x.transpose(1, 2) if tall else x
    p = (p * (1.0 - MUON["lr"] * MUON["weight_decay"]) - MUON["lr"] * _adjust(case) * x).to(t)
    torch._foreach_copy_(s["p"], list(p))
    torch._foreach_copy_(s["buf"], list(buf))
    return dict(p=s["p"], buf=s["buf"])


PLAIN = dict(embed=_embed, embed_bwd=_embed_bwd, rms=_rms, rms_bwd=_rms_bwd, muon=_muon)
OUTPUTS = dict(embed=("out",), embed_bwd=("dtable",), rms=("h", "y", "scales"), rms_bwd=("dx", "dweight"), muon=("p", "buf"))


def run(state):
    case = state["case"]
    if own:
        state["program"]()
        return {k: state[k] for k in OUTPUTS[case["op"]] if k in state}
    return PLAIN[case["op"]](state, case)


# ---- work -------------------------------------------------------------------------------------------------------------------
def work(case):
    es, op = ITEM[case["dtype"]], case["op"]
    if op in ("embed", "embed_bwd"):
        n, v, d = case["tokens"], case["vocab"], case["dim"]
        used = n - int(n * case["pad"])
        met = min(v, used)                                   # at most so many rows of the table are met
        if op == "embed":
            return dict(bytes=4 * n + es * d * (met + n), flops=n * d)
        return dict(bytes=4 * n + es * d * (used + (2 * met if case["accumulate"] else v)), flops=2 * used * d)
    if op in ("rms", "rms_bwd"):
        n, c = case["rows"], case["cols"]
        if op == "rms_bwd":
            return dict(bytes=es * (n * c * (4 if case["residual"] else 3) + 2 * c), flops=10 * n * c)
        out = n * c + 4 * n * -(-c // (case["group"] or c)) if case["quant"] else es * n * c
        return dict(bytes=es * (n * c * (3 if case["residual"] else 1) + c) + out, flops=6 * n * c)
    # a symmetric product needs half of its entries
    n, lo, hi = case["count"], min(case["rows"], case["cols"]), max(case["rows"], case["cols"])
    return dict(bytes=5 * es * n * lo * hi, flops=n * STEPS * (3.0 * lo * lo * hi + float(lo) ** 3))


# ---- 64 bits ----------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = _inputs(case, seed)
    t, op = DTYPES[case["dtype"]], case["op"]
    f = {k: v.double() for k, v in s.items() if torch.is_tensor(v) and v.is_floating_point()}
    if op in ("embed", "embed_bwd"):
        at = torch.nonzero((s["ids"] >= 0) & (s["ids"] < case["vocab"])).flatten()
        ids = s["ids"][at].long()
        if op == "embed":
            out = torch.zeros(case["tokens"], case["dim"], dtype=torch.float64, device="cuda")
            out[at] = f["table"].index_select(0, ids) * case["scale"]
            return dict(out=out)
        total = torch.zeros(case["vocab"], case["dim"], dtype=torch.float64, device="cuda").index_add_(0, ids, f["dout"][at], alpha=case["scale"])
        return dict(dtable=total + f["dtable"] if case["accumulate"] else total)
    if op == "rms":
        h = f["x"] + f["residual"] if case["residual"] else f["x"]
        y = f["weight"] * h / (h.square().sum(1, keepdim=True) / case["cols"] + RMS_EPS).sqrt()
        out = dict(h=h) if case["residual"] else {}
        if not case["quant"]:
            return dict(out, y=y)
        width = case["group"] or case["cols"]
        q, scales = torch.empty_like(y), []
        for lo in range(0, case["cols"], width):
            part = y[:, lo:lo + width]
            scale = part.abs().amax(1, keepdim=True).clamp_min(AMAX_FLOOR) / E4M3_MAX
            scales.append(scale)
            v = part / scale
            step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)       # 3 bits behind the leading one
            q[:, lo:lo + width] = torch.round(v / step) * step
        return dict(out, y=q.clamp(-E4M3_MAX, E4M3_MAX), scales=torch.cat(scales, 1))
    if op == "rms_bwd":
        n = case["cols"]
        norm = (f["h"].square().sum(1, keepdim=True) / n + RMS_EPS).sqrt()
        along = (f["dy"] * f["weight"] * f["h"]).sum(1, keepdim=True)
        dx = f["dy"] * f["weight"] / norm - f["h"] * along / (n * norm ** 3)
        return dict(dx=dx + f["dh"] if case["residual"] else dx, dweight=(f["dy"] * f["h"] / norm).sum(0))
    p_out, buf_out = [], []
    for p, g, buf in zip(s["p"], s["g"], s["buf"]):
        g, buf = g.double(), buf.double() * MUON["momentum"] + g.double()
        u = g + MUON["momentum"] * buf.to(t).double()        # the update reads the buffer as it is stored
        x = u / (torch.linalg.vector_norm(u) + NORM_EPS)
        for _ in range(STEPS):
            if x.shape[0] <= x.shape[1]:
                a = x @ x.T
                x = NS[0] * x + NS[1] * (a @ x) + NS[2] * (a @ (a @ x))
            else:
                a = x.T @ x
                x = NS[0] * x + NS[1] * (x @ a) + NS[2] * ((x @ a) @ a)
        p_out.append(p.double() * (1.0 - MUON["lr"] * MUON["weight_decay"]) - MUON["lr"] * _adjust(case) * x)
        buf_out.append(buf)
    return dict(p=p_out, buf=buf_out)
