# SPDX-License-Identifier: MPL-2.0
"""Cases of serving from a paged cache: several sequences in one batch, each with new tokens behind cached ones.

  rope       rows of heads rotated by positions of their own: pairs of a head's halves or neighbours, the whole head or its
             first part, frequencies scaled for long contexts
  norm_rope  RMSNorm of each head of q and k, and the rotation
  append     q rotated, k rotated and written with v into the pages of the cache (with the norms before, or without)
  attention  the new tokens' attention over the cached keys and their own, causal, with a window or without

A cache is [pages][2 (keys, values)][KV heads][page][head size]; sequence s has its new tokens in rows start[s] ..
start[s + 1] - 1 and, these included, len[s] keys in the pages that row s of the page table lists.
"""
import ctypes
import math
import random

import numpy as np
import torch

own = False

EPS = 1e-5
HEADS = {"135m": (9, 3, 64), "360m": (15, 5, 64), "wide": (32, 8, 128)}  # SmolLM2; a wider model: heads, KV heads, size


def listed():
    return [
        # one decode token's stacked q|k heads: the smallest call, where latency counts
        dict(name="rope_135m_1", family="rope", N=1, NH=12, HD=64, rot=64, layout="half", scaling="none", far=2048,
             type="f32"),
        # a batch of long prompts' heads, the first half of each rotated, neighbouring pairs, far positions
        dict(name="rope_4096x40x128_bf16", family="rope", N=4096, NH=40, HD=128, rot=64, layout="pairs", scaling="yarn",
             far=131072, type="bf16"),
        # a ragged batch of short prompts
        dict(name="norm_rope_360m_333_bf16", family="norm_rope", N=333, NH=15, NKV=5, HD=64, rot=64, layout="half",
             scaling="none", far=2048, type="bf16"),
        # long prompts in a wider model, fp32 products
        dict(name="norm_rope_wide_4096", family="norm_rope", N=4096, NH=32, NKV=8, HD=128, rot=128, layout="half",
             scaling="llama3", far=32768, type="f32"),
        # a decode step of eight sequences, fp32
        dict(name="append_360m_8", family="append", S=8, new=1, mix="even", ctx=2048, page=16, NH=15, NKV=5, HD=64, rot=64,
             layout="half", scaling="none", norm=False, type="f32", shape=1),
        # prompts' chunks of a ragged batch in a wider model, with the norms
        dict(name="append_wide_chunks_bf16", family="append", S=16, new=512, mix="ragged", ctx=2048, page=64, NH=32, NKV=8,
             HD=128, rot=128, layout="half", scaling="llama3", norm=True, type="bf16", shape=2),
        # one decode token over a short chat
        dict(name="attention_135m_1x300", family="attention", S=1, new=1, mix="even", ctx=300, page=16, NH=9, NKV=3, HD=64,
             window=0, type="f32", shape=3),
        # a decode step of 32 sequences of all lengths
        dict(name="attention_360m_32_bf16", family="attention", S=32, new=1, mix="even", ctx=2048, page=16, NH=15, NKV=5,
             HD=64, window=0, type="bf16", shape=4),
        # a decode step of 64 long sequences in a wider model: the cache is read from memory
        dict(name="attention_wide_64x8192_bf16", family="attention", S=64, new=1, mix="even", ctx=8192, page=64, NH=32,
             NKV=8, HD=128, window=0, type="bf16", shape=5),
        # a chunk of one prompt behind a cached part, fp32
        dict(name="attention_360m_512_of_4096", family="attention", S=1, new=512, mix="even", ctx=4096, page=32, NH=15,
             NKV=5, HD=64, window=0, type="f32", shape=6),
        # one chunk of a prompt beside the decode steps of the others, with a window
        dict(name="attention_360m_mixed_bf16", family="attention", S=24, new=333, mix="one", ctx=4096, page=16, NH=15,
             NKV=5, HD=64, window=1024, type="bf16", shape=7),
        # a large chunk of a long prompt in a wider model
        dict(name="attention_wide_2048_of_16384_bf16", family="attention", S=1, new=2048, mix="even", ctx=16384, page=64,
             NH=32, NKV=8, HD=128, window=0, type="bf16", shape=8),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    f = rng.choice(["rope", "norm_rope", "append", "append", "attention", "attention", "attention", "attention"])
    HD = rng.choice([64, 64, 128, 128, 80, 96, 256])
    NKV = rng.choice([1, 2, 3, 4, 5, 8])
    NH = NKV * rng.choice([1, 2, 3, 4, 7, 8])
    turn = dict(HD=HD, rot=rng.choice([HD, HD, HD // 2, HD // 4]), layout=rng.choice(["half", "pairs"]),
                scaling=rng.choice(["none", "linear", "llama3", "yarn"]))
    kind = rng.choice(["f32", "bf16"])
    if f == "rope":
        return dict(family=f, N=_log_int(rng, 1, min(8192, (20 << 20) // (NH * HD))), NH=NH, far=_log_int(rng, 64, 1 << 20),
                    type=kind, **turn)
    if f == "norm_rope":
        return dict(family=f, N=_log_int(rng, 1, min(8192, (20 << 20) // ((NH + NKV) * HD))), NH=NH, NKV=NKV,
                    far=_log_int(rng, 64, 1 << 20), type=kind, **turn)
    mix = rng.choice(["even", "one", "ragged"])
    page, shape = rng.choice([8, 16, 16, 32, 64, 128]), rng.randrange(1 << 30)
    if f == "append":
        ctx = _log_int(rng, 16, 4096)
        S = _log_int(rng, 1, max(1, min(128, (64 << 20) // (ctx * NKV * HD))))
        new = _log_int(rng, 1, max(1, min(ctx, (16 << 20) // (S * (NH + 2 * NKV) * HD))))
        return dict(family=f, S=S, new=new, mix=mix, ctx=ctx, page=page, NH=NH, NKV=NKV, norm=rng.random() < 0.5, type=kind,
                    shape=shape, **turn)
    ctx = _log_int(rng, 1, 32768)
    S = _log_int(rng, 1, max(1, min(128, (256 << 20) // (ctx * NKV * HD))))
    most = min(2048, ctx, (16 << 20) // (NH * HD * S), (1 << 30) // (S * NH * ctx), (1 << 36) // (S * NH * HD * ctx))
    new = 1 if rng.random() < 0.4 else _log_int(rng, 1, max(1, most))
    return dict(family=f, S=S, new=new, mix=mix, ctx=ctx, page=page, NH=NH, NKV=NKV, HD=HD,
                window=_log_int(rng, 1, ctx) if rng.random() < 0.25 else 0, type=kind, shape=shape)


# ---------------------------------------------------------------- inputs

def _lens(case):
    """New tokens and keys of each sequence, a function of the case alone."""
    rng, S, new, ctx = random.Random(case["shape"]), case["S"], case["new"], case["ctx"]
    if case["mix"] == "even":
        n = [new] * S
    elif case["mix"] == "one":
        n = [1] * S
        n[rng.randrange(S)] = new
    else:
        n = [rng.randint(1, new) for _ in range(S)]
    total = [max(k, rng.randint((ctx + 3) // 4, ctx)) for k in n]
    total[rng.randrange(S)] = ctx
    return n, total


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 2654435761 % (1 << 62) + 131)
    return g


def _kind(case):
    return torch.bfloat16 if case["type"] == "bf16" else torch.float32


def _randn(g, *shape, kind=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda").to(kind)


def _heads(g, n, heads, size, kind):
    """Rows of heads, some heads up to four times as large as others."""
    gain = 1 + 3 * torch.rand(heads, 1, generator=g, device="cuda")
    return (_randn(g, n, heads, size) * gain).to(kind).view(n, heads * size)


SCALED = dict(factor=8.0, low=1.0, high=4.0, original=8192.0)  # a context eight times the first one
THETA = 500000.0


def _batch(case, g, kind):
    """A cache whose pages are dealt out at random, and the tables of the batch."""
    n, total = _lens(case)
    page, S = case["page"], case["S"]
    need = [(t + page - 1) // page for t in total]
    width, count = max(need), sum(need) + 3
    cache = _randn(g, count, 2, case["NKV"], page, case["HD"], kind=kind)
    order = torch.randperm(count, generator=g, device="cuda").to(torch.int32)
    pages = torch.full((S, width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for s in range(S):
        pages[s, :need[s]] = order[at:at + need[s]]
        at += need[s]
    start = torch.tensor([sum(n[:s]) for s in range(S + 1)], dtype=torch.int32, device="cuda")
    return dict(cache=cache, pages=pages, start=start, len=torch.tensor(total, dtype=torch.int32, device="cuda"),
                N=sum(n), new=max(n), ctx=max(total), count=count, width=width)


def _inputs(case, seed):
    """The inputs as plain tensors, a function of (case, seed)."""
    g, kind, f, HD = _gen(seed), _kind(case), case["family"], case["HD"]
    if f in ("rope", "norm_rope"):
        N, NH = case["N"], case["NH"]
        pos = torch.randint(0, case["far"], (N,), generator=g, device="cuda", dtype=torch.int32)
        q = _heads(g, N, NH, HD, kind)
        if f == "rope":
            return dict(q=q, pos=pos)
        return dict(q=q, k=_heads(g, N, case["NKV"], HD, kind), pos=pos, gain=1 + 0.1 * _randn(g, 2, HD))
    b = _batch(case, g, kind)
    b["q"] = _heads(g, b["N"], case["NH"], HD, kind)
    if f == "append":
        b["k"], b["v"] = (_heads(g, b["N"], case["NKV"], HD, kind) for _ in range(2))
        b["gain"] = 1 + 0.1 * _randn(g, 2, HD)
    return b


# ---------------------------------------------------------------- the framework's calls

_backend = None


def _be():
    """The program's one backend context."""
    global _backend
    if _backend is None:
        import bmhip
        _backend = bmhip.Backend()
    return _backend


class _Shared:
    """The device memory of a backend buffer (backend_buffer_s starts with its device address, see
    include/backend_hip_device.h) in the form torch takes without a copy."""

    def __init__(self, buf, shape, typestr):
        ptr = ctypes.cast(buf.h, ctypes.POINTER(ctypes.c_void_p))[0]
        self.buf = buf
        self.__cuda_array_interface__ = dict(shape=tuple(shape), typestr=typestr, data=(ptr, False), version=3,
                                             strides=None)


_TYPES = {torch.float32: "<f4", torch.int32: "<i4", torch.bfloat16: "<i2"}


def _buffer(shape, dtype):
    """A backend buffer and a tensor over its memory."""
    n = math.prod(shape) * torch.empty(0, dtype=dtype).element_size()
    buf = _be().alloc(n)
    t = torch.as_tensor(_Shared(buf, shape, _TYPES[dtype]), device="cuda")
    return buf, t.view(dtype)


def _upload(values):
    """A backend buffer holding a tensor's values (the buffer's zero fill is over first), and a tensor over it."""
    buf, t = _buffer(values.shape, values.dtype)
    _be().synchronize()
    t.copy_(values)
    return buf, t


def _floats(*v):
    return _be().upload(np.float32(v))


class _Encoded:
    """The dispatches of one pass, bound once; each call encodes and commits them, and takes back the encoder of its
    previous call, so that a program keeps the GPU busy."""

    def __init__(self, calls):
        import bmhip
        be = _be()
        self.lib, self.keep, self.args, self.enc = bmhip.lib(), calls, [], None
        for name, bufs, grid in calls:
            n = len(bufs)
            arr = (ctypes.c_void_p * n)(*[b.h for b in bufs])
            self.args.append((be.kernel(name).h, arr, None, n, grid, 1, 1, 256, 1, 1))

    def __call__(self):
        lib = self.lib
        if self.enc:
            lib.backend_encode_wait_timed(self.enc)
        enc = lib.backend_encode_begin(_be().ctx)
        for a in self.args:
            if lib.backend_encode_dispatch(enc, *a) != 0:
                raise RuntimeError("dispatch rejected")
        lib.backend_encode_commit(enc)
        self.enc = enc

    def __del__(self):
        if self.enc and _be().ctx:
            self.lib.backend_encode_wait_timed(self.enc)
            self.enc = None


def _turns(case):
    """The table of the rotation's turns a position, as a program builds it once for a model, and the rotation's factor."""
    import bmhip
    table, mscale = bmhip.rope_turns(case["rot"], THETA, case["scaling"], **SCALED)
    return _be().upload(table), mscale


def _bind(case, i):
    """The pass's dispatches over backend buffers, and its outputs."""
    f, kind, HD, NH = case["family"], _kind(case), case["HD"], case["NH"]
    suffix, par = "_bf16" if case["type"] == "bf16" else "", _be().params
    q = _upload(i["q"])[0]
    qo, qt = _buffer(i["q"].shape, kind)
    if f != "attention":
        turns, mscale = _turns(case)
        pairs = int(case["layout"] == "pairs")
    if f == "rope":
        N = case["N"]
        return _Encoded([("rope_forward_rows" + suffix, [
            q, qo, _upload(i["pos"])[0], turns, par(N, NH, HD, case["rot"], pairs, NH * HD, NH * HD), _floats(mscale)], N)]
        ), dict(q=qt)
    NKV = case["NKV"]
    QW, KW = NH * HD, NKV * HD
    if f == "norm_rope":
        N = case["N"]
        ko, kt = _buffer(i["k"].shape, kind)
        return _Encoded([("qk_norm_rope_forward" + suffix, [
            q, _upload(i["k"])[0], qo, ko, _upload(i["pos"])[0], turns, _upload(i["gain"])[0],
            par(N, NH, NKV, HD, case["rot"], pairs, QW, KW, QW, KW), _floats(mscale, EPS)], N)]), dict(q=qt, k=kt)
    (cache, ct), N, S = _upload(i["cache"]), i["N"], case["S"]
    start, length, pages = (_upload(i[k])[0] for k in ("start", "len", "pages"))
    if f == "append":
        return _Encoded([("kv_append_paged" + suffix, [
            q, _upload(i["k"])[0], _upload(i["v"])[0], qo, cache, start, length, pages, turns, _upload(i["gain"])[0],
            par(N, S, NH, NKV, HD, case["rot"], pairs, QW, KW, KW, QW, case["page"], i["count"], i["width"],
                int(case["norm"])), _floats(mscale, EPS)], N)]), dict(q=qt, cache=ct)
    return _Encoded([("attention_forward_paged" + suffix, [
        q, cache, qo, start, length, pages, par(N, S, NH, NKV, HD, QW, QW, case["page"], i["count"], i["width"], 1,
                                                case["window"]), _floats(HD ** -0.5)], N)]), dict(out=qt)


def prepare(case, seed):
    i = _inputs(case, seed)
    if own:  # the framework's kernels take the backend's own buffers
        call, out = _bind(case, i)
        torch.cuda.synchronize()
        return dict(call=call, out=out)
    return dict(i, case=case, kind=_kind(case))


# ---------------------------------------------------------------- the plain forms

def _frequencies(rot, scaling):
    """Radians a position of each pair, in 64 bits, and the factor of the rotated part."""
    i = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    f = THETA ** (-2 * i / rot)
    factor, low, high, original = (SCALED[k] for k in ("factor", "low", "high", "original"))
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "llama3":  # waves longer than original / low slowed down, shorter than original / high not, between them mixed
        waves = original * f / (2 * math.pi)
        mix = ((waves - low) / (high - low)).clamp(0, 1)
        return f * (mix + (1 - mix) / factor), 1.0
    if scaling == "yarn":  # the pairs between `high` and `low` waves over the original context are mixed by their number
        pair = [rot * math.log(original / (w * 2 * math.pi)) / (2 * math.log(THETA)) for w in (high, low)]
        first, last = max(math.floor(pair[0]), 0), min(math.ceil(pair[1]), rot - 1)
        mix = ((i - first) / max(last - first, 0.001)).clamp(0, 1)
        return f * (1 - mix + mix / factor), 0.1 * math.log(factor) + 1
    return f, 1.0


def _rotate(x, pos, case):
    """Rows of heads [n][heads][size] in fp32, rotated by pos."""
    rot = case["rot"]
    f, m = _frequencies(rot, case["scaling"])
    angle = pos.double()[:, None, None] * f
    c, s = (torch.cos(angle) * m).float(), (torch.sin(angle) * m).float()
    y = x.clone()
    if case["layout"] == "half":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y[..., :rot // 2], y[..., rot // 2:rot] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., :rot:2], x[..., 1:rot:2]
        y[..., :rot:2], y[..., 1:rot:2] = a * c - b * s, b * c + a * s
    return y


def _turned(x, pos, case, gain=None):
    y = x.float().view(x.shape[0], -1, case["HD"])
    if gain is not None:
        y = y * torch.rsqrt(y.square().mean(dim=-1, keepdim=True) + EPS) * gain
    return _rotate(y, pos, case)


def _places(s):
    """Sequence and position of each new token."""
    n = s["start"].long()
    row = torch.arange(s["N"], device="cuda")
    seq = torch.searchsorted(n, row, right=True) - 1
    return seq, row - n[seq + 1] + s["len"][seq]


def _attend(s, case):
    """Sequences padded to the longest: scores of all of a sequence's rows and keys, softmax, sum."""
    S, NH, NKV, HD, page = (case[k] for k in ("S", "NH", "NKV", "HD", "page"))
    R, n, L = NH // NKV, s["new"], s["ctx"]
    start, length = s["start"].long(), s["len"].long()
    count = start[1:] - start[:-1]
    i, j = torch.arange(n, device="cuda"), torch.arange(L, device="cuda")
    row = (start[:-1, None] + i).clamp(max=s["N"] - 1)
    pos = (length - count)[:, None] + i
    seen = (j <= pos[..., None]) & (i < count[:, None])[..., None]
    if case["window"]:
        seen &= j > pos[..., None] - case["window"]
    kv = s["cache"][s["pages"].long()[:, j // page].clamp(min=0), :, :, j % page].float()
    k, v = kv[:, :, 0].permute(0, 2, 3, 1).contiguous(), kv[:, :, 1].permute(0, 2, 1, 3).contiguous()
    q = s["q"].float()[row].view(S, n, NKV, R, HD).permute(0, 2, 3, 1, 4).reshape(S, NKV, R * n, HD)
    w = torch.matmul(q, k).view(S, NKV, R, n, L) * HD ** -0.5
    seen = seen[:, None, None]
    w = torch.where(seen, w, -math.inf)
    top = w.amax(dim=-1, keepdim=True)
    w = torch.exp(w - torch.where(torch.isfinite(top), top, 0.0))
    total = w.sum(dim=-1, keepdim=True)
    o = torch.matmul(w.view(S, NKV, R * n, L), v).view(S, NKV, R, n, HD)
    o = torch.where(total > 0, o / total, 0.0)
    out = torch.empty_like(s["q"])
    kept = i < count[:, None]
    out[row[kept]] = o.permute(0, 3, 1, 2, 4)[kept].reshape(-1, NH * HD).to(out.dtype)
    return out


def run(s):
    if own:
        s["call"]()
        return s["out"]
    case, kind = s["case"], s["kind"]
    f = case["family"]
    if f == "rope":
        return dict(q=_turned(s["q"], s["pos"], case).to(kind).view(s["q"].shape))
    if f == "norm_rope":
        q, k = (_turned(s[x], s["pos"], case, s["gain"][n]).to(kind).view(s[x].shape) for n, x in enumerate("qk"))
        return dict(q=q, k=k)
    if f == "attention":
        return dict(out=_attend(s, case))
    seq, pos = _places(s)
    gains = s["gain"] if case["norm"] else (None, None)
    q, k = (_turned(s[x], pos, case, gains[n]).to(kind) for n, x in enumerate("qk"))
    page, cache = s["pages"][seq, pos // case["page"]].long(), s["cache"]
    cache[page, 0, :, pos % case["page"]] = k
    cache[page, 1, :, pos % case["page"]] = s["v"].view(k.shape)
    return dict(q=q.view(s["q"].shape), cache=cache)


# ---------------------------------------------------------------- work

def work(case):
    f, e, HD, NH = case["family"], 2 if case["type"] == "bf16" else 4, case["HD"], case["NH"]
    if f in ("rope", "norm_rope"):
        n = case["N"] * (NH + case.get("NKV", 0)) * HD
        return dict(bytes=2 * n * e + 4 * case["N"], flops=n * (3 if f == "rope" else 7))
    n, total = _lens(case)
    N, NKV, tables = sum(n), case["NKV"], 4 * (2 * case["S"] + sum(-(-t // case["page"]) for t in total))
    if f == "append":
        return dict(bytes=2 * N * (NH + 2 * NKV) * HD * e + tables, flops=N * (NH + NKV) * HD * (7 if case["norm"] else 3))
    w = case["window"] or max(total)
    pairs = sum(min(p + 1, w) for a, t in zip(n, total) for p in range(t - a, t))
    keys = sum(min(t, w + a - 1) for a, t in zip(n, total))
    return dict(bytes=2 * N * NH * HD * e + 2 * keys * NKV * HD * e + tables, flops=4 * pairs * NH * HD)


# ---------------------------------------------------------------- the same in 64 bits

def _exact_turned(x, pos, case, gain=None):
    """The rotation as products with e^(i angle)."""
    rot, size = case["rot"], case["HD"]
    x = x.double().reshape(len(pos), -1, size)
    if gain is not None:
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / size + EPS) * gain.double()
    m, table = 1.0, []
    for i in range(rot // 2):
        w = THETA ** (-2.0 * i / rot)
        if case["scaling"] == "linear":
            w /= SCALED["factor"]
        elif case["scaling"] == "llama3":
            length = 2 * math.pi / w
            if length > SCALED["original"] / SCALED["low"]:
                w /= SCALED["factor"]
            elif length > SCALED["original"] / SCALED["high"]:
                part = (SCALED["original"] / length - SCALED["low"]) / (SCALED["high"] - SCALED["low"])
                w = (1 - part) * w / SCALED["factor"] + part * w
        elif case["scaling"] == "yarn":
            def border(waves):
                return rot * math.log(SCALED["original"] / (2 * math.pi * waves)) / math.log(THETA) / 2
            a, b = max(0, math.floor(border(SCALED["high"]))), min(rot - 1, math.ceil(border(SCALED["low"])))
            part = min(1.0, max(0.0, (i - a) / max(b - a, 0.001)))
            w, m = w / SCALED["factor"] * part + w * (1 - part), 1 + math.log(SCALED["factor"]) / 10
        table.append(w)
    angle = torch.outer(pos.double(), torch.tensor(table, dtype=torch.float64, device="cuda"))[:, None]
    turn = torch.polar(torch.full_like(angle, m), angle)
    h = rot // 2
    z = torch.complex(x[..., :h], x[..., h:rot]) if case["layout"] == "half" else torch.view_as_complex(
        x[..., :rot].reshape(*x.shape[:-1], h, 2).contiguous())
    z = z * turn
    z = torch.cat([z.real, z.imag], -1) if case["layout"] == "half" else torch.view_as_real(z).flatten(-2)
    return torch.cat([z, x[..., rot:]], -1).reshape(len(pos), -1)


def exact(case, seed):
    i, f = _inputs(case, seed), case["family"]
    if f == "rope":
        return dict(q=_exact_turned(i["q"], i["pos"], case))
    if f == "norm_rope":
        return dict(q=_exact_turned(i["q"], i["pos"], case, i["gain"][0]),
                    k=_exact_turned(i["k"], i["pos"], case, i["gain"][1]))
    n, total = _lens(case)
    page, NH, NKV, HD = (case[k] for k in ("page", "NH", "NKV", "HD"))
    slots = [(i["pages"][s, torch.arange(t, device="cuda") // page].long() * page
              + torch.arange(t, device="cuda") % page) for s, t in enumerate(total)]  # page * size + place of each key
    if f == "append":
        pos = torch.cat([torch.arange(t - a, t, device="cuda") for a, t in zip(n, total)])
        slot = torch.cat([x[t - a:] for a, t, x in zip(n, total, slots)])
        gain = i["gain"] if case["norm"] else (None, None)
        flat = i["cache"].double().permute(0, 3, 1, 2, 4).reshape(-1, 2, NKV, HD)
        flat[slot, 0] = _exact_turned(i["k"], pos, case, gain[1]).view(-1, NKV, HD)
        flat[slot, 1] = i["v"].double().view(-1, NKV, HD)
        return dict(q=_exact_turned(i["q"], pos, case, gain[0]),
                    cache=flat.view(-1, page, 2, NKV, HD).permute(0, 2, 3, 1, 4).contiguous())
    out = torch.zeros(i["N"], NH, HD, dtype=torch.float64, device="cuda")
    at = 0
    for a, t, x in zip(n, total, slots):
        p = torch.arange(t - a, t, device="cuda")[:, None]
        j = torch.arange(t, device="cuda")[None]
        hide = (j > p) | (j <= p - case["window"] if case["window"] else torch.zeros_like(j > p))
        for g in range(NKV):
            k, v = (i["cache"][x // page, b, g, x % page].double() for b in (0, 1))
            for h in range(g * (NH // NKV), (g + 1) * (NH // NKV)):
                w = (i["q"][at:at + a, h * HD:(h + 1) * HD].double() @ k.T / math.sqrt(HD)).masked_fill(hide, -math.inf)
                out[at:at + a, h] = torch.softmax(w, dim=-1) @ v
        at += a
    return dict(out=out.view(i["N"], NH * HD))
