"""What the operators around given tokens are measured on: the log probabilities of tokens with
entropy and alternatives, from stored logits (``token_scores``) and from the rows before the head
(``LmHead.score``), and the arrays that tell a packed step of unequal sequences where its tokens lie
(``kernels.step_index``, ``kernels.map_pages``).

``listed`` names the cases, ``draw`` gives more of the same ranges, ``prepare`` makes what a program
has in hand, ``run`` is one pass (the plain form by elementary torch operations, or the library's own
calls), ``work`` what a pass cannot do without, ``exact`` the answer in 64 bits.
"""
import functools
import math
import random

import torch

own = False

DEV = "cuda:0"
PAGE = 64                 # positions of a cache page
VOCAB = 151936            # the measured models' vocabulary
CONTEXT = 40960           # and their longest sequence
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


# ---------------------------------------------------------------------------- the cases
def listed():
    return [
        # one user who asks for five alternatives beside every token of the answer
        dict(name="token_b1_top5", kind="token", rows=1, vocab=VOCAB, top=5, masked=0.0),
        # a server's full batch with twenty alternatives each
        dict(name="token_b64_top20", kind="token", rows=64, vocab=VOCAB, top=20, masked=0.0),
        # a batch whose grammar leaves few tokens, an odd vocabulary, log probabilities alone
        dict(name="token_b37_masked", kind="token", rows=37, vocab=50257, top=0, masked=0.97),
        # the logits of a long prompt that a program kept
        dict(name="token_2048_top5", kind="token", rows=2048, vocab=VOCAB, top=5, masked=0.0),
        # one answer of 24 tokens scored on a small model's head
        dict(name="head_24_short", kind="head", rows=24, width=1024, vocab=VOCAB, top=5,
             dtype="bfloat16", cap=0.0),
        # a multiple-choice question's answers together, twenty alternatives
        dict(name="head_333_top20", kind="head", rows=333, width=4096, vocab=VOCAB, top=20,
             dtype="bfloat16", cap=0.0),
        # a prompt of 2,048 tokens on the 8B model's head: what perplexity asks for
        dict(name="head_2048", kind="head", rows=2048, width=4096, vocab=VOCAB, top=5,
             dtype="bfloat16", cap=0.0),
        # a head with capped logits, odd in rows and vocabulary
        dict(name="head_1001_cap", kind="head", rows=1001, width=2048, vocab=100003, top=0,
             dtype="bfloat16", cap=30.0),
        # the true 32-bit path
        dict(name="head_f32_200", kind="head", rows=200, width=1024, vocab=VOCAB, top=5,
             dtype="float32", cap=0.0),
        # a first step of a few questions
        dict(name="index_4", kind="index", count=4, lo=30, hi=200, past=0, ring=0),
        # 64 unequal prompts in one step
        dict(name="index_64", kind="index", count=64, lo=16, hi=495, past=2000, ring=0),
        # a large step over layers with a window, whose pages form rings
        dict(name="index_700_ring", kind="index", count=700, lo=1, hi=373, past=9000, ring=81),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(("token", "token", "head", "head", "head_f32", "index"))
    top = rng.choice((0, 1, 5, 20, rng.randint(0, 32)))
    if kind == "token":
        return dict(kind="token", rows=_log_int(rng, 1, 2048),
                    vocab=rng.choice((VOCAB, 32768, _log_int(rng, 1000, VOCAB))), top=top,
                    masked=rng.choice((0.0, 0.0, 0.9)))
    if kind == "head":
        width = rng.choice((1024, 2048, 4096, 8 * rng.randint(32, 512)))
        return dict(kind="head", rows=_log_int(rng, 1, 2048), width=width,
                    vocab=rng.choice((VOCAB, 32768, _log_int(rng, 1000, VOCAB))), top=top,
                    dtype="bfloat16", cap=rng.choice((0.0, 0.0, 30.0)))
    if kind == "head_f32":
        return dict(kind="head", rows=_log_int(rng, 1, 400), width=8 * rng.randint(32, 128),
                    vocab=rng.choice((VOCAB, _log_int(rng, 1000, VOCAB))), top=top,
                    dtype="float32", cap=0.0)
    count = _log_int(rng, 1, 1000)
    hi = _log_int(rng, 2, min(8000, 131072 // count))
    return dict(kind="index", count=count, lo=rng.randint(1, hi), hi=hi,
                past=rng.choice((0, _log_int(rng, 1, 20000))), ring=rng.choice((0, 0, rng.randint(2, 150))))


def spread(lo, hi, n):
    """``n`` whole numbers from ``lo`` to ``hi`` in even steps, in an order of no account."""
    out = [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]
    random.Random(n).shuffle(out)
    return out


# ---------------------------------------------------------------------------- inputs
class Values:
    """Seeded values on the device, drawn in the order in which they are asked for."""

    def __init__(self, seed):
        self.gen = torch.Generator(device=DEV)
        self.gen.manual_seed(seed)

    def normal(self, shape, std):
        return torch.empty(shape, dtype=torch.float32, device=DEV).normal_(0.0, std, generator=self.gen)

    def grid(self, shape, std, step, dtype):
        """A bell whose values are whole multiples of ``step`` (a power of two), at most 255 of them,
        as weights and rows hold that went through 8 bits. A sum of products of such values is the
        same in every order, so which logit is the greater is a matter of the inputs alone."""
        t = self.normal(shape, std / step).round_().clamp_(-255, 255)
        return t.mul_(step).to(dtype)

    def ids(self, shape, below):
        return torch.randint(0, below, shape, generator=self.gen, device=DEV)

    def share(self, shape):
        return torch.rand(shape, generator=self.gen, device=DEV)


def _token_inputs(case, seed):
    """Logits as a trained model gives them: a broad bell and a few tokens far above it; under a
    grammar most are minus infinity. Half of the given tokens are the likeliest of their row."""
    v = Values(seed)
    rows, vocab = case["rows"], case["vocab"]
    logits = v.normal((rows, vocab), 2.2)
    n = 40
    at = v.ids((rows, n), vocab // n) + torch.arange(n, device=DEV) * (vocab // n)
    logits.scatter_add_(1, at, 2.0 + 12.0 * v.share((rows, n)))
    if case["masked"]:
        logits.masked_fill_(v.share((rows, vocab)) < case["masked"], -math.inf)
    best = v.share((rows,)) < 0.5
    tokens = torch.where(best, logits.argmax(1), v.ids((rows,), vocab)).to(torch.int32)
    return logits, tokens


def _head_inputs(case, seed):
    v = Values(seed)
    dtype = DTYPES[case["dtype"]]
    h = v.grid((case["rows"], case["width"]), 1.0, 2.0 ** -5, dtype)
    weight = v.grid((case["vocab"], case["width"]), 1.5 / math.sqrt(case["width"]), 2.0 ** -10, dtype)
    return h, weight, v.ids((case["rows"],), case["vocab"]).to(torch.int32)


def _index_inputs(case, seed):
    """Which slots take part, what they hold, what they bring, the pages that they hold and the free
    ones, and the page table of all slots."""
    v = Values(seed)
    B, ring = case["count"], case["ring"]
    slots = torch.randperm(B + B // 4 + 1, generator=v.gen, device=DEV)[:B]
    past = torch.tensor(spread(0, case["past"], B), device=DEV)
    new = torch.tensor(spread(case["lo"], case["hi"], B), device=DEV)
    held, need = (past + PAGE - 1) // PAGE, (past + new + PAGE - 1) // PAGE
    if ring:
        held, need = held.clamp(max=ring), need.clamp(max=ring)
    n = int((need - held).sum())
    pages = torch.randperm(n + 1000, generator=v.gen, device=DEV)[:n]
    table = v.ids((B + B // 4 + 1, ring or CONTEXT // PAGE), n + 1000)
    i32 = lambda t: t.to(torch.int32)
    return i32(slots), i32(past), i32(new), i32(held), i32(pages), i32(table)


@functools.lru_cache(maxsize=None)
def _runtime(dtype):
    """What a program's models of one type share: the device's scratch and error word."""
    from mormot2_ai_b200 import Runtime
    return Runtime(DTYPES[dtype], DEV)


def prepare(case, seed):
    s = {"case": case}
    if case["kind"] == "token":
        s["logits"], s["tokens"] = _token_inputs(case, seed)
    elif case["kind"] == "head":
        s["h"], s["weight"], s["tokens"] = _head_inputs(case, seed)
        if own:
            # the bound part that a model keeps: it names the weight and lays nothing out
            from mormot2_ai_b200 import PartSpec
            from mormot2_ai_b200.parts import HEADS
            s["head"] = HEADS.build(PartSpec("lm_head", {
                "name": "head", "tied": False, "vocab_size": case["vocab"],
                "hidden_size": case["width"], "softcap": case["cap"]}))
            s["head"].bind({"head": s["weight"]}, _runtime(case["dtype"]))
    else:
        s["slots"], s["past"], s["new"], s["held"], s["pages"], s["table"] = _index_inputs(case, seed)
        T = int(s["new"].sum())
        s["T"], s["N"] = T, s["pages"].numel()
        s["tok_seq"], s["tok_pos"], s["tok_slot"] = (
            torch.zeros(T, dtype=torch.int32, device=DEV) for _ in range(3))
        s["seq_start"] = torch.zeros(case["count"] + 1, dtype=torch.int32, device=DEV)
    return s


# ---------------------------------------------------------------------------- run
def _plain_scores(x, tokens, top, order=None):
    """x [rows, vocab] float32. ``order``: what the alternatives are ordered by (x itself)."""
    m = x.amax(1, keepdim=True)
    d = x - m
    e = d.exp()
    total = e.sum(1, keepdim=True)
    logz = total.log()
    given = d.gather(1, tokens.long()[:, None]) - logz
    # e d is 0 where a token is masked out
    entropy = logz[:, 0] - (e * d.clamp(min=-1e30)).sum(1) / total[:, 0]
    if not top:
        return [given[:, 0], entropy]
    # one whole number a value: its place among the floats first, the lowest id first among equals
    bits = ((x if order is None else order) + 0.0).view(torch.int32)
    place = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    vocab = x.shape[1]
    key = place * 2 ** 32 + (vocab - 1 - torch.arange(vocab, device=x.device))
    ids = vocab - 1 - (key.topk(top, dim=1).values & 0xFFFFFFFF)
    return [given[:, 0], entropy, ids.to(torch.int32), d.gather(1, ids) - logz]


def _plain_index(s):
    slots, past, new, held = (s[k].long() for k in ("slots", "past", "new", "held"))
    B = slots.numel()
    which = torch.arange(B, device=DEV)
    ends = new.cumsum(0)
    s["seq_start"][1:] = ends
    seq = torch.repeat_interleave(which, new, output_size=s["T"])
    s["tok_seq"][:] = seq
    s["tok_pos"][:] = torch.arange(s["T"], device=DEV) - (ends - new)[seq] + past[seq]
    s["tok_slot"][:] = slots[seq]
    need = (past + new + PAGE - 1) // PAGE
    if s["case"]["ring"]:
        need = need.clamp(max=s["case"]["ring"])
    more = need - held
    seq = torch.repeat_interleave(which, more, output_size=s["N"])
    entry = torch.arange(s["N"], device=DEV) - (more.cumsum(0) - more)[seq] + held[seq]
    s["table"][slots[seq], entry] = s["pages"]


def run(s):
    case = s["case"]
    if case["kind"] == "token":
        if own:
            from mormot2_ai_b200 import token_scores
            got = token_scores(s["logits"], s["tokens"], top=case["top"])
        else:
            return _plain_scores(s["logits"], s["tokens"], case["top"])
    elif case["kind"] == "head":
        if own:
            got = s["head"].score(s["h"], s["tokens"], top=case["top"])
        else:
            raw = s["h"].float() @ s["weight"].float().t()
            if case["cap"]:
                return _plain_scores(case["cap"] * torch.tanh(raw / case["cap"]), s["tokens"],
                                     case["top"], raw)
            return _plain_scores(raw, s["tokens"], case["top"])
    else:
        if own:
            from mormot2_ai_b200 import kernels as K
            K.step_index(s["slots"], s["past"], s["new"], s["seq_start"], s["tok_seq"],
                         s["tok_pos"], s["tok_slot"])
            K.map_pages(s["table"], s["slots"], s["past"], s["new"], s["held"], s["pages"],
                        case["ring"])
        else:
            _plain_index(s)
        return [s[k] for k in ("seq_start", "tok_seq", "tok_pos", "tok_slot", "table")]
    out = [got.logprobs, got.entropy]
    return out + [got.top_ids, got.top_logprobs] if case["top"] else out


# ---------------------------------------------------------------------------- work
def work(case):
    if case["kind"] == "index":
        B, ring = case["count"], case["ring"]
        past, new = spread(0, case["past"], B), spread(case["lo"], case["hi"], B)
        up = lambda n: min(-(-n // PAGE), ring) if ring else -(-n // PAGE)
        N = sum(up(p + n) - up(p) for p, n in zip(past, new))
        return {"bytes": 16 * B + 4 * (B + 1) + 12 * sum(new) + 8 * N, "flops": sum(new) + N}
    rows, vocab = case["rows"], case["vocab"]
    ends = rows * (4 + 8 + 8 * case["top"])
    if case["kind"] == "token":
        return {"bytes": 4 * rows * vocab + ends, "flops": 6 * rows * vocab}
    size, width = DTYPES[case["dtype"]].itemsize, case["width"]
    return {"bytes": size * width * (vocab + rows) + ends, "flops": 2 * rows * vocab * width}


# ---------------------------------------------------------------------------- exact
def _exact_rows(x, tokens, top, raw):
    """x [rows, vocab] float64: every quantity from the probabilities themselves."""
    logp = x - torch.logsumexp(x, dim=1, keepdim=True)
    p = logp.exp()
    entropy = -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(1)
    out = [logp[torch.arange(x.shape[0], device=x.device), tokens.long()], entropy]
    if top:
        ids = raw.sort(dim=1, descending=True, stable=True).indices[:, :top]
        out.append(torch.gather(logp, 1, ids))
    return out


def exact(case, seed):
    if case["kind"] == "index":
        return None            # whole numbers
    if case["kind"] == "token":
        logits, tokens = _token_inputs(case, seed)
        rows_of = lambda a, b: logits[a:b].double()
    else:
        h, weight, tokens = _head_inputs(case, seed)
        wide = weight.double().t()
        rows_of = lambda a, b: h[a:b].double() @ wide
    cap, parts = case.get("cap", 0.0), []
    for a in range(0, case["rows"], 128):
        raw = rows_of(a, a + 128)
        x = cap * torch.tanh(raw / cap) if cap else raw
        parts.append(_exact_rows(x, tokens[a:a + 128], case["top"], raw))
    got = [torch.cat(p) for p in zip(*parts)]
    return [got[0], got[1], None, got[2]] if case["top"] else got
