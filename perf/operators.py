"""Cases for the operators between a classifier's logits and its weights: log probabilities of given classes with entropy and top
alternatives, their gradient, the global gradient norm with clipping, and the momentum update with the clip factor applied.

`run` computes them in elementary torch operations, or, where `own` is true, through the framework's entry points."""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
CODES = {"f32": 0, "f16": 1, "bf16": 2}
I32 = 3

# weights and biases of the nin-cifar10 net, in its order
NIN = [14400, 192, 30720, 160, 15360, 96, 460800, 192, 36864, 192, 36864, 192, 331776, 192, 36864, 192, 1920, 10]


def listed():
    return [
        # the test pass of a ten-class net over one minibatch (nin-cifar10): latency
        dict(name="logprob_10x128_f32", op="logprob", layout="class", type="f32", classes=10, cases=128, pad=0, top=5, entropy=True, masked=0.0),
        # a thousand classes, one minibatch, the top five that such nets report
        dict(name="logprob_1000x128_f32", op="logprob", layout="class", type="f32", classes=1000, cases=128, pad=0, top=5, entropy=True, masked=0.0),
        # one token of one sequence while it is generated, with the alternatives a server reports
        dict(name="logprob_1x131072_bf16", op="logprob", layout="case", type="bf16", classes=131072, cases=1, pad=0, top=20, entropy=True, masked=0.0),
        # odd vocabulary, odd batch, padded rows, classes that a grammar forbids: no alternatives asked for
        dict(name="logprob_257x50021_f16", op="logprob", layout="case", type="f16", classes=50021, cases=257, pad=27, top=0, entropy=True, masked=0.3),
        # scoring prompts: many positions over a large vocabulary
        dict(name="logprob_2048x131072_bf16", op="logprob", layout="case", type="bf16", classes=131072, cases=2048, pad=0, top=20, entropy=True, masked=0.0),
        # training step of a thousand-class net
        dict(name="grad_1000x128_f32", op="grad", layout="class", type="f32", classes=1000, cases=128, pad=0, entropy=False, logz=False),
        # odd sizes, with an entropy bonus and a penalty on the normaliser
        dict(name="grad_511x50021_f32", op="grad", layout="case", type="f32", classes=50021, cases=511, pad=0, entropy=True, logz=True),
        # training step over a large vocabulary
        dict(name="grad_2048x131072_bf16", op="grad", layout="case", type="bf16", classes=131072, cases=2048, pad=0, entropy=False, logz=True),
        # the gradients of the nin-cifar10 net
        dict(name="clip_nin_f32", op="clip", sizes="nin", tensors=18, total=0, type="f32", out="f32", packed=False, loss_scale=1.0, share=0.5),
        # half-precision gradients of a large net in many tensors of any size, unscaled and clipped into float32
        dict(name="clip_300t_256m_bf16", op="clip", sizes="mixed", tensors=300, total=1 << 28, type="bf16", out="f32", packed=True, loss_scale=1024.0, share=0.1),
        # the update of the nin-cifar10 net
        dict(name="update_nin_f32", op="update", sizes="nin", tensors=18, total=0, share=0.5),
        # the update of a large net
        dict(name="update_120t_128m_f32", op="update", sizes="mixed", tensors=120, total=1 << 27, share=0.1),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["logprob", "logprob", "grad", "grad", "clip", "update"])
    if op in ("logprob", "grad"):
        classes = _log_int(rng, 2, 200000)
        cases = _log_int(rng, 1, max(1, min(8192, (1 << 27) // classes)))
        case = dict(op=op, layout=rng.choice(["class", "case"]), type=rng.choice(["f32", "f16", "bf16"]), classes=classes, cases=cases,
                    pad=rng.choice([0, 0, 1, 13, 64]))
        if op == "logprob":
            return dict(case, top=min(classes, rng.choice([0, 1, 5, 20, 32])), entropy=rng.random() < 0.7, masked=rng.choice([0.0, 0.0, 0.3, 0.9]))
        return dict(case, entropy=rng.random() < 0.4, logz=rng.random() < 0.4)
    tensors = _log_int(rng, 1, 400)
    if op == "clip":
        kind = rng.choice(["f32", "f16", "bf16"])
        return dict(op=op, sizes="mixed", tensors=tensors, total=_log_int(rng, 1000, 1 << 27), type=kind, out=rng.choice([kind, "f32"]),
                    packed=rng.random() < 0.5, loss_scale=rng.choice([1.0, 256.0]), share=rng.choice([0.05, 0.5, 2.0]))
    return dict(op=op, sizes="mixed", tensors=tensors, total=_log_int(rng, 1000, 1 << 26), share=rng.choice([0.05, 0.5, 2.0]))


# ---------------------------------------------------------------- what both sides are given
def _sizes(case):
    if case["sizes"] == "nin":
        return NIN
    rng = random.Random(case["tensors"] * 7919 + case["total"])
    shares = [math.exp(rng.gauss(0.0, 1.5)) for _ in range(case["tensors"])]
    return [max(1, int(case["total"] * s / sum(shares))) for s in shares]


def _offsets(sizes, unit):
    offsets, at = [], 0
    for n in sizes:
        offsets.append(at)
        at += -(-n // unit) * unit
    return offsets, at


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) % (1 << 62))


def _logits(case, gen):
    """Logits and labels as a user has them: a dense or padded matrix, class-major (float labels) or case-major (int32 labels)."""
    V, N, dtype = case["classes"], case["cases"], TYPES[case["type"]]
    rows, cols = (V, N) if case["layout"] == "class" else (N, V)
    store = torch.randn(rows, cols + case["pad"], generator=gen, device="cuda", dtype=torch.float32).mul_(2.5)
    x = store[:, :cols]
    labels = torch.randint(0, V, (N,), generator=gen, device="cuda", dtype=torch.int64)
    by_case = x.t() if case["layout"] == "class" else x
    at = torch.arange(N, device="cuda")
    if case.get("masked", 0.0) > 0.0:
        by_case.masked_fill_(torch.rand(by_case.shape, generator=gen, device="cuda") < case["masked"], float("-inf"))
    by_case[at, labels] = torch.rand(N, generator=gen, device="cuda").mul_(16.0)      # some predictions are sure, some are not
    labels = torch.where(torch.rand(N, generator=gen, device="cuda") < 0.05, torch.full_like(labels, -1), labels)   # no class: padding
    return store.to(dtype)[:, :cols], labels.to(torch.float32 if case["layout"] == "class" else torch.int32)


def _kernels():
    if "mckernels" in sys.modules:      # a program imports it once
        return sys.modules["mckernels"]
    folder = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cuda-convnet_amd")
    here = os.path.join(os.getcwd(), "cuda-convnet_amd")
    folder = here if os.path.isdir(here) else folder
    if folder not in sys.path:
        sys.path.insert(0, folder)
    import mckernels
    return mckernels


def _upload(array):
    return torch.from_numpy(np.frombuffer(bytes(array), dtype=np.uint8).copy()).cuda()


def prepare(case, seed):
    gen = _generator(seed)
    state = dict(case)
    if case["op"] in ("logprob", "grad"):
        N = case["cases"]
        x, labels = _logits(case, gen)
        state.update(logits=x, labels=labels, class_stride=x.stride(0) if case["layout"] == "class" else 1,
                     case_stride=1 if case["layout"] == "class" else x.stride(0))
        if case["op"] == "logprob":
            state.update(logp=torch.empty(N, device="cuda"), stats=torch.empty(2, N, device="cuda"),
                         H=torch.empty(N, device="cuda") if case["entropy"] else None,
                         top_classes=torch.empty(case["top"], N, device="cuda", dtype=torch.int32),
                         top_logp=torch.empty(case["top"], N, device="cuda"))
            if own:
                size = _kernels().lib().mc_log_probs_workspace_bytes(CODES[case["type"]], state["class_stride"], state["case_stride"], N, case["classes"], case["top"])
                state.update(work=torch.empty(max(16, size), device="cuda", dtype=torch.uint8), work_bytes=size)
        else:
            logp, stats, H = _forward(x, labels, case["layout"])[:3]
            g = torch.randn(3, N, generator=gen, device="cuda").div_(N)
            state.update(stats=stats, H=H, g_logp=g[0].abs().neg().contiguous(), g_H=g[1].mul(0.1).contiguous(), g_z=g[2].abs().mul(0.01).contiguous(),
                         target=torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device="cuda"))
        return state
    sizes = _sizes(case)
    if case["op"] == "clip":
        offsets, whole = _offsets(sizes, 1 if case["packed"] else 64)
        grads = torch.randn(whole, generator=gen, device="cuda").mul_(0.01 * case["loss_scale"]).to(TYPES[case["type"]])
        out = torch.empty(whole, device="cuda", dtype=TYPES[case["out"]])
        out.zero_()
        state.update(flat_grad=grads, flat_out=out, grads=[grads[o:o + n] for o, n in zip(offsets, sizes)], outs=[out[o:o + n] for o, n in zip(offsets, sizes)],
                     scale=1.0 / case["loss_scale"], stats=torch.empty(2, device="cuda"),
                     max_norm=case["share"] * 0.01 * math.sqrt(sum(sizes)))
        if own:
            mk = _kernels()
            spans = mk.grad_spans([(g.data_ptr(), o.data_ptr(), g.numel(), state["scale"], CODES[case["type"]], CODES[case["out"]])
                                   for g, o in zip(state["grads"], state["outs"])])
            state.update(spans=_upload(spans), num_spans=len(spans))
    else:
        offsets, whole = _offsets(sizes, 64)
        weights, inc, grads = (torch.randn(whole, generator=gen, device="cuda").mul_(s) for s in (0.05, 1e-4, 1e-3))
        rates = [0.05 if i % 2 == 0 else 0.1 for i in range(len(sizes))]          # weights and biases learn at rates of their own
        decay = [-0.0005 * r if i % 2 == 0 else 0.0 for i, r in enumerate(rates)]
        state.update(weights=weights, inc=inc, flat_grad=grads, offsets=offsets, sizes=sizes, rates=rates, decay=decay, momentum=0.9,
                     stats=torch.empty(2, device="cuda"), max_norm=case["share"] * 0.015 * math.sqrt(sum(sizes)))
        if own:
            mk = _kernels()
            spans = mk.grad_spans([(grads.data_ptr() + 4 * o, 0, n, 1.0 / r, CODES["f32"], CODES["f32"]) for o, n, r in zip(offsets, sizes, rates)])
            steps = np.array([(o + at, min(4096, n - at), 0.9, d, 0) for o, n, d in zip(offsets, sizes, decay) for at in range(0, n, 4096)],
                             dtype=[("start", "<u8"), ("count", "<u4"), ("mom", "<f4"), ("wceps", "<f4"), ("pad", "<u4")])
            state.update(spans=_upload(spans), num_spans=len(spans), steps=_upload(steps.tobytes()), num_steps=len(steps))
    if own:
        size = mk.lib().mc_grad_norm_workspace_bytes(state["num_spans"])
        state.update(work=torch.empty(max(16, size), device="cuda", dtype=torch.uint8), work_bytes=size)
    return state


# ---------------------------------------------------------------- the plain forms
def _forward(x, labels, layout):
    """Log probability of each case's label (0 where it is no class), (max, log of the sum), entropy, and the shifted logits."""
    xf = x.float()
    dim = 0 if layout == "class" else 1
    m = xf.amax(dim, keepdim=True)
    d = xf - m
    e = d.exp()
    s = e.sum(dim, keepdim=True)
    log_s = s.log()
    p = e / s
    H = -torch.where(p > 0, p * (d - log_s), torch.zeros_like(p)).sum(dim)
    index = labels.long()
    valid = (index >= 0) & (index < x.shape[dim])
    picked = d.gather(dim, index.clamp(0, x.shape[dim] - 1).unsqueeze(dim)).squeeze(dim) - log_s.squeeze(dim)
    stats = torch.stack([m.squeeze(dim), log_s.squeeze(dim)])
    return torch.where(valid, picked, torch.zeros_like(picked)), stats, H, d


def _plain_logprob(s):
    logp, stats, H, d = _forward(s["logits"], s["labels"], s["layout"])
    out = {"logp": logp, "stats": stats}
    if s["entropy"]:
        out["entropy"] = H
    if s["top"]:
        dim = 0 if s["layout"] == "class" else 1
        bits = (s["logits"].float() + 0.0).view(torch.int32).long()
        order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)
        classes = torch.arange(s["classes"], device="cuda").unsqueeze(1 - dim)
        keys = (order << 32) | (0x7FFFFFFF - classes)          # ties go to the lowest class
        best = 0x7FFFFFFF - (keys.topk(s["top"], dim=dim).values & 0xFFFFFFFF)
        top = d.gather(dim, best) - stats[1].unsqueeze(dim)
        best = torch.where(top == float("-inf"), torch.full_like(best, -1), best)
        out["top_classes"] = (best if dim == 0 else best.t()).to(torch.int32).contiguous()
        out["top_logp"] = (top if dim == 0 else top.t()).contiguous()
    return out


def _plain_grad(s):
    x, dim = s["logits"].float(), 0 if s["layout"] == "class" else 1
    logp = (x - s["stats"][0].unsqueeze(dim)) - s["stats"][1].unsqueeze(dim)
    p = logp.exp()
    index = s["labels"].long()
    valid = (index >= 0) & (index < s["classes"])
    g = torch.where(valid, s["g_logp"], torch.zeros_like(s["g_logp"]))
    dx = p * (s["g_z"] - g if s["logz"] else -g).unsqueeze(dim)
    if s["entropy"]:
        dx = dx - torch.where(p > 0, p * (logp + s["H"].unsqueeze(dim)), torch.zeros_like(p)) * s["g_H"].unsqueeze(dim)
    dx.scatter_add_(dim, index.clamp(0, s["classes"] - 1).unsqueeze(dim), g.unsqueeze(dim))
    return {"grad": dx.to(s["logits"].dtype)}


def _factor(square, max_norm):
    norm = square.sqrt()
    return torch.stack([norm, (max_norm / norm).clamp(max=1.0)]).float()


def _plain_clip(s):
    square = torch.stack([(g.double() * s["scale"]).square().sum() for g in s["grads"]]).sum()
    stats = _factor(square, s["max_norm"])
    f = stats[1] * s["scale"]
    [o.copy_(g.float() * f) for g, o in zip(s["grads"], s["outs"])]
    return {"stats": stats, "out": s["flat_out"]}


def _update_tensor(s, f, at, n, decay):
    w, inc, g = (s[k][at:at + n] for k in ("weights", "inc", "flat_grad"))
    inc.mul_(s["momentum"]).add_(g * f)
    if decay:
        inc.add_(w * decay)
    w.add_(inc)


def _plain_update(s):
    square = torch.stack([(s["flat_grad"][o:o + n].double() / r).square().sum() for o, n, r in zip(s["offsets"], s["sizes"], s["rates"])]).sum()
    stats = _factor(square, s["max_norm"])
    [_update_tensor(s, stats[1], o, n, d) for o, n, d in zip(s["offsets"], s["sizes"], s["decay"])]
    return {"stats": stats, "weights": s["weights"], "inc": s["inc"]}


# ---------------------------------------------------------------- the framework's calls
def _ptr(t):
    return t.data_ptr() if t is not None and t.numel() else None


def _own_logprob(s, call, stream):
    label_type = CODES["f32"] if s["layout"] == "class" else I32
    call("mc_log_probs", _ptr(s["logits"]), CODES[s["type"]], s["class_stride"], s["case_stride"], _ptr(s["labels"]), label_type, s["cases"], s["classes"],
         _ptr(s["logp"]), _ptr(s["H"]), _ptr(s["stats"]), _ptr(s["top_classes"]), _ptr(s["top_logp"]), s["top"], _ptr(s["work"]), s["work_bytes"], stream)
    out = {"logp": s["logp"], "stats": s["stats"]}
    if s["entropy"]:
        out["entropy"] = s["H"]
    if s["top"]:
        out.update(top_classes=s["top_classes"], top_logp=s["top_logp"])
    return out


def _own_grad(s, call, stream):
    label_type = CODES["f32"] if s["layout"] == "class" else I32
    call("mc_log_probs_grad", _ptr(s["logits"]), CODES[s["type"]], s["class_stride"], s["case_stride"], _ptr(s["labels"]), label_type, s["cases"], s["classes"],
         _ptr(s["stats"]), _ptr(s["H"]) if s["entropy"] else None, _ptr(s["g_logp"]), 1.0, _ptr(s["g_H"]), 1.0 if s["entropy"] else 0.0,
         _ptr(s["g_z"]), 1.0 if s["logz"] else 0.0, _ptr(s["target"]), s["class_stride"], s["case_stride"], 0, stream)
    return {"grad": s["target"]}


def _own_clip(s, call, stream):
    call("mc_grad_norm", _ptr(s["spans"]), s["num_spans"], s["max_norm"], _ptr(s["stats"]), _ptr(s["work"]), s["work_bytes"], stream)
    call("mc_clip_grads", _ptr(s["spans"]), s["num_spans"], _ptr(s["stats"]), stream)
    return {"stats": s["stats"], "out": s["flat_out"]}


def _own_update(s, call, stream):
    call("mc_grad_norm", _ptr(s["spans"]), s["num_spans"], s["max_norm"], _ptr(s["stats"]), _ptr(s["work"]), s["work_bytes"], stream)
    call("mc_weights_update_spans_clipped", _ptr(s["weights"]), _ptr(s["inc"]), _ptr(s["flat_grad"]), _ptr(s["steps"]), s["num_steps"], _ptr(s["stats"]), stream)
    return {"stats": s["stats"], "weights": s["weights"], "inc": s["inc"]}


def run(state):
    if own:
        forms = {"logprob": _own_logprob, "grad": _own_grad, "clip": _own_clip, "update": _own_update}
        return forms[state["op"]](state, _kernels().call, torch.cuda.current_stream().cuda_stream)
    return {"logprob": _plain_logprob, "grad": _plain_grad, "clip": _plain_clip, "update": _plain_update}[state["op"]](state)


def work(case):
    """Each input read once and each output written once."""
    if case["op"] in ("logprob", "grad"):
        V, N, size = case["classes"], case["cases"], BYTES[case["type"]]
        if case["op"] == "logprob":
            return {"bytes": V * N * size + N * (4 + 4 + 8 + (4 if case["entropy"] else 0) + 8 * case["top"]), "flops": V * N * (6 if case["entropy"] else 4)}
        return {"bytes": 2 * V * N * size + N * (16 + (8 if case["entropy"] else 0) + (4 if case["logz"] else 0)), "flops": V * N * (7 if case["entropy"] else 4)}
    E = sum(_sizes(case))
    if case["op"] == "clip":
        return {"bytes": E * (BYTES[case["type"]] + BYTES[case["out"]]), "flops": 4 * E}
    return {"bytes": 20 * E, "flops": 9 * E}


# ---------------------------------------------------------------- the definitions, in 64 bits
def _exact_rows(x, labels, top):
    """One block of cases, case-major, in 64 bits."""
    x = x.double()
    z = torch.logsumexp(x, 1)
    logp = x - z.unsqueeze(1)
    H = torch.special.entr(logp.exp()).sum(1)
    y = labels.long()
    ok = (y >= 0) & (y < x.shape[1])
    picked = torch.where(ok, logp[torch.arange(len(y), device=x.device), y.clamp(0, x.shape[1] - 1)], torch.zeros_like(z))
    m = x.max(1).values
    best = None
    if top:
        values, classes = torch.sort(logp, dim=1, descending=True, stable=True)
        best = (torch.where(values[:, :top].isinf(), torch.full_like(classes[:, :top], -1), classes[:, :top]).to(torch.int32), values[:, :top])
    return logp, z, H, picked, m, ok, best


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("logprob", "grad"):
        x = s["logits"].t() if case["layout"] == "class" else s["logits"]
        step = max(1, (1 << 25) // case["classes"])
        blocks = []
        for a in range(0, case["cases"], step):
            b = slice(a, a + step)
            logp, z, H, picked, m, ok, best = _exact_rows(x[b], s["labels"][b], case.get("top", 0))
            if case["op"] == "logprob":
                blocks.append((picked, torch.stack([m, z - m]), H) + (best or ()))
                continue
            # of the inputs that the call is given: the normaliser and the entropy of the forward pass, as they were rounded
            logp = x[b].double() - (s["stats"][0, b].double() + s["stats"][1, b].double()).unsqueeze(1)
            p = logp.exp()
            g = torch.where(ok, s["g_logp"][b].double(), torch.zeros_like(z))
            dx = -g.unsqueeze(1) * p
            dx[torch.arange(len(g), device="cuda"), s["labels"][b].long().clamp(0, case["classes"] - 1)] += g
            if case["logz"]:
                dx += s["g_z"][b].double().unsqueeze(1) * p
            if case["entropy"]:
                dx -= s["g_H"][b].double().unsqueeze(1) * torch.where(p > 0, p * (logp + s["H"][b].double().unsqueeze(1)), torch.zeros_like(p))
            blocks.append((dx,))
        if case["op"] == "grad":
            dx = torch.cat([b[0] for b in blocks])
            return {"grad": dx.t() if case["layout"] == "class" else dx}
        out = {"logp": torch.cat([b[0] for b in blocks]), "stats": torch.cat([b[1] for b in blocks], 1)}
        if case["entropy"]:
            out["entropy"] = torch.cat([b[2] for b in blocks])
        if case["top"]:
            out["top_classes"] = torch.cat([b[3] for b in blocks]).t().contiguous()
            out["top_logp"] = torch.cat([b[4] for b in blocks]).t().contiguous()
        return out
    if case["op"] == "clip":
        norm = math.sqrt(sum(float(torch.sum((g.double() * s["scale"]) ** 2)) for g in s["grads"]))
        factor = min(1.0, s["max_norm"] / norm)
        out = torch.zeros(s["flat_out"].shape, dtype=torch.float64, device="cuda")
        base = s["flat_grad"].data_ptr()
        for g in s["grads"]:
            at = (g.data_ptr() - base) // g.element_size()
            out[at:at + g.numel()] = g.double() * (factor * s["scale"])
        return {"stats": torch.tensor([norm, factor], dtype=torch.float64), "out": out}
    g = s["flat_grad"].double()
    norm = math.sqrt(sum(float(torch.sum((g[o:o + n] / r) ** 2)) for o, n, r in zip(s["offsets"], s["sizes"], s["rates"])))
    factor = min(1.0, s["max_norm"] / norm)
    weights, inc = s["weights"].double(), s["inc"].double()
    for o, n, d in zip(s["offsets"], s["sizes"], s["decay"]):
        inc[o:o + n] = s["momentum"] * inc[o:o + n] + factor * g[o:o + n] + d * weights[o:o + n]
        weights[o:o + n] += inc[o:o + n]
    return {"stats": torch.tensor([norm, factor], dtype=torch.float64), "weights": weights, "inc": inc}
