"""The vocabulary-sized losses: what is measured of them, and their plain forms.

Three operators of a language model's last layer, over N rows (tokens) and a vocabulary of V words:

* ``linear_cross_entropy``: softmax cross entropy of ``x [N, D] @ weight [V, D]^T + bias`` against one
  target a row, with its gradients, without keeping the logits;
* ``linear_topk_distill``: the same head against a teacher's top logits;
* ``topk_distill``: logits that the caller has, against a teacher's top logits.

``own`` false computes the plain forms below, true makes the calls of ``determined_1_amd.ops.vocab_loss``.
"""
import torch

own = False

IGNORE = -100
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # the log-probability of the one token that a user or a tool proposes next: latency, one read of the head
        {"name": "score_one_token", "op": "ce", "train": False, "dtype": "bf16", "rows": 1, "dim": 4096, "vocab": 128000,
         "keep": 1.0, "bias": False, "smooth": 0.0, "reduction": "none", "scale": 1.0},
        # log-probabilities of a prompt or an answer (perplexity, ranking of choices), an odd vocabulary
        {"name": "score_prompt", "op": "ce", "train": False, "dtype": "bf16", "rows": 700, "dim": 2048, "vocab": 50021,
         "keep": 1.0, "bias": False, "smooth": 0.0, "reduction": "none", "scale": 1.0},
        # masked-language-model step at the shape of the BERT benchmark: 12 sequences of 384, 15 % of the tokens are targets
        {"name": "train_masked_lm", "op": "ce", "train": True, "dtype": "bf16", "rows": 4608, "dim": 768, "vocab": 30522,
         "keep": 0.15, "bias": True, "smooth": 0.0, "reduction": "mean", "scale": 1.0},
        # the word-level recurrent language model's decoder: 35 steps of 64 sequences, 850 wide, fp32
        {"name": "train_word_lm", "op": "ce", "train": True, "dtype": "fp32", "rows": 2240, "dim": 850, "vocab": 10000,
         "keep": 1.0, "bias": True, "smooth": 0.0, "reduction": "mean", "scale": 1.0},
        # a translation or summary step: label smoothing, padded targets, sizes that divide by nothing, a loss scale
        {"name": "train_smoothed", "op": "ce", "train": True, "dtype": "fp16", "rows": 1003, "dim": 1111, "vocab": 20011,
         "keep": 0.8, "bias": True, "smooth": 0.1, "reduction": "sum", "scale": 16.0},
        # pretraining of a large causal model: two sequences of 4096 against a 128 k vocabulary
        {"name": "train_causal_lm", "op": "ce", "train": True, "dtype": "bf16", "rows": 8192, "dim": 4096, "vocab": 128000,
         "keep": 1.0, "bias": False, "smooth": 0.0, "reduction": "mean", "scale": 1.0},
        # a student's training step against 64 stored teacher logits a token
        {"name": "distill_head", "op": "head", "train": True, "dtype": "bf16", "rows": 2048, "dim": 2048, "vocab": 32000,
         "keep": 0.9, "bias": False, "top": 64, "pad": 0.0, "temperature": 2.0, "reduction": "mean", "scale": 1.0},
        # a small student in fp32, lists of other lengths
        {"name": "distill_head_fp32", "op": "head", "train": True, "dtype": "fp32", "rows": 333, "dim": 768, "vocab": 30522,
         "keep": 1.0, "bias": True, "top": 20, "pad": 0.3, "temperature": 1.0, "reduction": "sum", "scale": 1.0},
        # a few rows of logits: launches and latency
        {"name": "distill_few_rows", "op": "logits", "train": True, "dtype": "fp32", "rows": 8, "vocab": 32000,
         "keep": 1.0, "top": 16, "pad": 0.0, "temperature": 1.0, "reduction": "mean", "scale": 1.0},
        # a validation pass
        {"name": "distill_eval", "op": "logits", "train": False, "dtype": "fp32", "rows": 512, "vocab": 30522,
         "keep": 1.0, "top": 32, "pad": 0.2, "temperature": 2.0, "reduction": "none", "scale": 1.0},
        # ragged lists, rows without a list, an odd vocabulary, a loss scale
        {"name": "distill_ragged", "op": "logits", "train": True, "dtype": "fp16", "rows": 1777, "vocab": 50021,
         "keep": 0.7, "top": 100, "pad": 0.4, "temperature": 3.0, "reduction": "sum", "scale": 16.0},
        # a training step on whole logits of a large vocabulary
        {"name": "distill_large", "op": "logits", "train": True, "dtype": "bf16", "rows": 4096, "vocab": 128000,
         "keep": 1.0, "top": 64, "pad": 0.0, "temperature": 2.0, "reduction": "sum", "scale": 1.0},
    ]


def _log_uniform(rng, low, high):
    return int(round(low * (high / low) ** rng.random()))


def draw(rng):
    op = rng.choice(["ce", "ce", "head", "logits", "logits"])
    case = {"op": op, "train": rng.random() < 0.75, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]),
            "rows": _log_uniform(rng, 1, 8192), "vocab": _log_uniform(rng, 1000, 128000),
            "keep": rng.choice([1.0, 1.0, 0.8, 0.5, 0.15]), "reduction": rng.choice(["mean", "sum", "none"])}
    if op != "logits":
        case["dim"] = _log_uniform(rng, 64, 4096)
        if rng.random() < 0.6:  # most models have a width of whole blocks
            case["dim"] = max(64, case["dim"] // 64 * 64)
        case["bias"] = rng.random() < 0.5
        while case["rows"] * case["dim"] * case["vocab"] > (2.0e11 if case["dtype"] == "fp32" else 1.0e12):
            case["rows"] = max(1, case["rows"] // 2)
    else:
        while case["rows"] * case["vocab"] * SIZE[case["dtype"]] > 1.0e9:
            case["rows"] = max(1, case["rows"] // 2)
    if op == "ce":
        case["smooth"] = rng.choice([0.0, 0.0, 0.1])
    else:
        case["top"] = _log_uniform(rng, 1, 128)
        case["pad"] = rng.choice([0.0, 0.0, 0.3])
        case["temperature"] = rng.choice([1.0, 2.0, 3.5])
    # half floats under a mean need the loss scale that their users have
    case["scale"] = 1.0 if case["dtype"] != "fp16" else 16.0 if case["reduction"] != "mean" else 16.0 * case["rows"]
    return case


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dev, dtype, rows, vocab = torch.device("cuda"), TYPES[case["dtype"]], case["rows"], case["vocab"]
    state = {"case": case}

    def normal(*shape, std=1.0, to=dtype):
        return torch.randn(*shape, generator=gen, device=dev).mul_(std).to(to)

    keep = torch.rand(rows, generator=gen, device=dev) < case["keep"]
    if case["keep"] < 1.0:
        keep[0] = True
    if case["op"] == "logits":
        state["logits"] = normal(rows, vocab, std=2.0)
    else:
        state["x"] = normal(rows, case["dim"])
        state["weight"] = normal(vocab, case["dim"], std=1.5 / case["dim"] ** 0.5)
        state["bias"] = normal(vocab, std=0.2) if case["bias"] else None
    if case["op"] == "ce":
        target = torch.randint(0, vocab, (rows,), generator=gen, device=dev)
        state["target"] = torch.where(keep, target, torch.full_like(target, IGNORE))
    else:
        top = case["top"]
        first = torch.randint(0, vocab, (rows, 1), generator=gen, device=dev)
        step = torch.randint(1, vocab // top + 1, (rows, 1), generator=gen, device=dev)
        index = (first + step * torch.arange(top, device=dev)) % vocab  # no word twice
        there = torch.rand(rows, top, generator=gen, device=dev) >= case["pad"]
        there[:, 0] = True
        state["index"] = torch.where(there & keep[:, None], index, torch.full_like(index, -1))
        state["teacher"] = normal(rows, top, std=3.0).sort(dim=1, descending=True).values
    if case["train"]:
        state["seed_grad"] = (torch.full((), case["scale"], device=dev) if case["reduction"] != "none"
                              else torch.rand(rows, generator=gen, device=dev).add_(0.5).mul_(case["scale"]))
    return state


def _reduce(case, rows, kept):
    """The loss and the derivative of it for each row's."""
    if case["reduction"] == "none":
        return rows, kept.to(rows.dtype)
    each = kept.to(rows.dtype)
    if case["reduction"] == "mean":
        each = each / kept.sum().clamp(min=1).to(rows.dtype)
    return (rows * each).sum(), each


def _plain(state):
    case = state["case"]
    head = case["op"] != "logits"
    if head:
        x, weight = state["x"].float(), state["weight"].float()
        z = x @ weight.t()
        if state["bias"] is not None:
            z = z + state["bias"].float()
    else:
        z = state["logits"].float()
    heat = case.get("temperature", 1.0)
    if heat != 1.0:
        z = z / heat
    high = z.max(dim=1, keepdim=True).values
    lse = (z - high).exp().sum(dim=1, keepdim=True).log() + high
    if case["op"] == "ce":
        smooth = case["smooth"]
        kept = state["target"] != IGNORE
        at = torch.where(kept, state["target"], torch.zeros_like(state["target"]))[:, None]
        share = torch.full(at.shape, 1.0 - smooth, device=z.device)
        rows = lse[:, 0] - (1.0 - smooth) * z.gather(1, at)[:, 0]
        if smooth:
            rows = rows - smooth * z.mean(dim=1)
    else:
        smooth = 0.0
        there = state["index"] >= 0
        kept = there.any(dim=1)
        at = torch.where(there, state["index"], torch.zeros_like(state["index"]))
        t = torch.where(there, state["teacher"].float() / heat, torch.full_like(state["teacher"].float(), float("-inf")))
        t = torch.where(kept[:, None], t, torch.zeros_like(t))
        t = t - t.max(dim=1, keepdim=True).values
        log_share = t - t.exp().sum(dim=1, keepdim=True).log()
        share = torch.where(there, log_share.exp(), torch.zeros_like(t))
        each = torch.where(there, share * (log_share - (z.gather(1, at) - lse)), torch.zeros_like(t))
        rows = heat * heat * each.sum(dim=1)
    rows = torch.where(kept, rows, torch.zeros_like(rows))
    loss, weigh = _reduce(case, rows, kept)
    out = {"loss": loss}
    if case["train"]:
        dz = (z - lse).exp()
        if smooth:
            dz = dz - smooth / case["vocab"]
        dz = dz.scatter_add_(1, at, -share)
        dz = dz * (weigh * state["seed_grad"] * heat)[:, None]
        if head:
            out["dx"] = (dz @ weight).to(state["x"].dtype)
            out["dweight"] = (dz.t() @ x).to(state["weight"].dtype)
            if state["bias"] is not None:
                out["dbias"] = dz.sum(dim=0).to(state["bias"].dtype)
        else:
            out["dlogits"] = dz.to(state["logits"].dtype)
    return out


def _own(state):
    from determined_1_amd.ops import vocab_loss

    case, train = state["case"], state["case"]["train"]
    names = ["logits"] if case["op"] == "logits" else ["x", "weight"] + (["bias"] if case["bias"] else [])
    leaf = {n: state[n].detach().requires_grad_(train) for n in names}
    if case["op"] == "ce":
        loss = vocab_loss.linear_cross_entropy(leaf["x"], leaf["weight"], state["target"], leaf.get("bias"), ignore_index=IGNORE,
                                               label_smoothing=case["smooth"], reduction=case["reduction"])
    elif case["op"] == "head":
        loss = vocab_loss.linear_topk_distill(leaf["x"], leaf["weight"], state["teacher"], state["index"], leaf.get("bias"),
                                              temperature=case["temperature"], reduction=case["reduction"])
    else:
        loss = vocab_loss.topk_distill(leaf["logits"], state["teacher"], state["index"], temperature=case["temperature"],
                                       reduction=case["reduction"])
    out = {"loss": loss.detach()}
    if train:
        grads = torch.autograd.grad(loss, list(leaf.values()), state["seed_grad"])
        out.update({"d" + n: g for n, g in zip(names, grads)})
    return out


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    size, rows, vocab = SIZE[case["dtype"]], case["rows"], case["vocab"]
    kept = max(1, round(rows * case["keep"]))
    lists = rows * (8 if case["op"] == "ce" else case["top"] * (8 + size)) + 4 * (rows if case["reduction"] == "none" else 1)
    if case["op"] == "logits":  # rows without a list need no read, but zeros are written for them
        return {"bytes": lists + size * vocab * (kept + (rows if case["train"] else 0)), "flops": kept * vocab * (7 if case["train"] else 4)}
    dim = case["dim"]
    head = size * (vocab * dim + (vocab if case["bias"] else 0))
    if not case["train"]:
        return {"bytes": lists + head + size * kept * dim, "flops": 2 * kept * vocab * dim}
    return {"bytes": lists + 2 * head + size * (kept + rows) * dim, "flops": 6 * kept * vocab * dim}


def exact(case, seed):
    """From the definition in 64 bits, row block by row block: the loss is the cross entropy (or the divergence) of
    two distributions, and its derivative by a logit is the difference of the two."""
    state = prepare(case, seed)
    f64, vocab, rows = torch.float64, case["vocab"], case["rows"]
    heat = case.get("temperature", 1.0)
    if case["op"] == "ce":
        kept = state["target"] != IGNORE
    else:
        kept = (state["index"] >= 0).any(dim=1)
    count = int(kept.sum())
    weigh = kept.to(f64) / (max(count, 1) if case["reduction"] == "mean" else 1)
    if case["op"] != "logits":
        weight = state["weight"].to(f64)
        bias = state["bias"].to(f64) if state["bias"] is not None else None
        dweight, dbias = torch.zeros_like(weight), torch.zeros(vocab, dtype=f64, device=weight.device)
    losses, by_row = [], []
    block = max(1, int(2e8) // vocab)
    for lo in range(0, rows, block):
        part = slice(lo, min(rows, lo + block))
        k = kept[part]
        if case["op"] == "logits":
            z = state["logits"][part].to(f64)
        else:
            x = state["x"][part].to(f64)
            z = torch.mm(x, weight.t().contiguous())
            if bias is not None:
                z += bias
        logp = torch.log_softmax(z / heat, dim=1)
        q = torch.zeros_like(z)
        if case["op"] == "ce":
            at = state["target"][part].clamp(min=0)[:, None]
            q.scatter_(1, at, 1.0 - case["smooth"])
            q += case["smooth"] / vocab
            loss = -(q * logp).sum(dim=1)
        else:
            index = state["index"][part]
            t = (state["teacher"][part].to(f64) / heat).masked_fill(index < 0, -float("inf"))
            t[~k] = 0.0
            share = torch.softmax(t, dim=1).masked_fill(index < 0, 0.0)
            q.scatter_add_(1, index.clamp(min=0), share)
            loss = (torch.xlogy(share, share).sum(dim=1) - (q * logp).sum(dim=1)) * heat * heat
        losses.append(torch.where(k, loss, torch.zeros_like(loss)))
        if case["train"]:
            seed_grad = state["seed_grad"].to(f64)
            up = weigh[part] * (seed_grad if seed_grad.dim() == 0 else seed_grad[part])
            dz = (logp.exp() - q) * (heat * up)[:, None]
            if case["op"] == "logits":
                by_row.append(dz)
            else:
                by_row.append(torch.mm(dz, weight))
                dweight += torch.mm(dz.t().contiguous(), x)
                dbias += dz.sum(dim=0)
    loss = torch.cat(losses)
    out = {"loss": loss if case["reduction"] == "none" else (loss * weigh).sum()}
    if case["train"]:
        if case["op"] == "logits":
            out["dlogits"] = torch.cat(by_row)
        else:
            out["dx"], out["dweight"] = torch.cat(by_row), dweight
            if bias is not None:
                out["dbias"] = dbias
    return out
