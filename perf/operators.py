# SPDX-License-Identifier: MPL-2.0
"""Cases of the 8-bit integer path: activations with one scale a token, weights with one scale an output channel.

  quantize  rows of a matrix to 8-bit codes with a scale each (weights at a model's load, tokens that no other kernel
            quantizes), and the values they stand for
  norm      a branch's output added to the residual stream, RMSNorm, and the result in 8-bit codes with a scale a token
  swiglu    SwiGLU of the gate and up products, in 8-bit codes with a scale a token
  matmul    tokens' codes times channels' codes, summed exactly, with both scales and a bias
  mlp       the four as a decoder layer's MLP uses them: norm, gate|up product, SwiGLU, down product

Codes are whole numbers of -127 .. 127; rows of codes lie `ld` bytes apart, a multiple of 16. Each pass that makes codes
returns the values they stand for (code times scale, in bf16) and the scales.
"""
import ctypes
import math

import numpy as np
import torch

own = False

EPS = 1e-5
DIMS = {"135m": (576, 1536), "360m": (960, 2560)}  # SmolLM2: width, MLP width


def listed():
    return [
        # the LM head's channels quantized at load
        dict(name="quantize_head_360m", family="quantize", M=49152, C=960, src="f32"),
        # attention outputs of a ragged batch, a width that is no multiple of 16
        dict(name="quantize_517x1001_bf16", family="quantize", M=517, C=1001, src="bf16"),
        # one decode token's norm: the smallest call, where latency counts
        dict(name="norm_135m_1", family="norm", N=1, C=576, src="f32"),
        # a short prompt's norm behind a product that wrote bf16
        dict(name="norm_360m_333_bf16", family="norm", N=333, C=960, src="bf16"),
        # a batch of long prompts in a wider model
        dict(name="norm_8192x4096", family="norm", N=8192, C=4096, src="f32"),
        # a short prompt's SwiGLU over separate fp32 products
        dict(name="swiglu_360m_333", family="swiglu", N=333, H=2560, src="f32"),
        # a long prompt's SwiGLU over one stacked gate|up product in bf16
        dict(name="swiglu_4096x8192_bf16", family="swiglu", N=4096, H=8192, src="bf16"),
        # one decode token's stacked gate and up projections
        dict(name="matmul_360m_gateup_1", family="matmul", M=1, C=960, OC=5120, out="f32", bias=False),
        # eight sequences' LM head
        dict(name="matmul_360m_head_8", family="matmul", M=8, C=960, OC=49152, out="f32", bias=False),
        # a ragged prompt through an odd shape, with a bias
        dict(name="matmul_777x2500x1999", family="matmul", M=777, C=2500, OC=1999, out="f32", bias=True),
        # a large product of long prompts, bf16 out for the next kernel
        dict(name="matmul_4096x4096x8192", family="matmul", M=4096, C=4096, OC=8192, out="bf16", bias=False),
        # a layer's MLP over a 512-token prompt
        dict(name="mlp_360m_512", family="mlp", model="360m", N=512),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """Half of the widths are multiples of 64, the others anything."""
    c = _log_int(rng, lo, hi)
    return max(64, c // 64 * 64) if rng.random() < 0.5 else c


def draw(rng):
    f = rng.choice(["quantize", "norm", "swiglu", "matmul", "matmul", "mlp"])
    src = rng.choice(["f32", "bf16"])
    if f == "quantize":
        C = _width(rng, 64, 8192)
        return dict(family=f, M=_log_int(rng, 1, min(65536, (32 << 20) // C)), C=C, src=src)
    if f == "norm":
        C = _width(rng, 64, 8192)
        return dict(family=f, N=_log_int(rng, 1, min(8192, (32 << 20) // C)), C=C, src=src)
    if f == "swiglu":
        H = _width(rng, 64, 16384)
        return dict(family=f, N=_log_int(rng, 1, min(4096, (32 << 20) // H)), H=H, src=src)
    if f == "matmul":
        C, OC = _width(rng, 64, 8192), _width(rng, 1, 16384)
        return dict(family=f, M=_log_int(rng, 1, max(1, min(4096, (4096 * 4096 * 8192) // (C * OC)))), C=C, OC=OC,
                    out=src, bias=rng.random() < 0.5)
    return dict(family=f, model=rng.choice(["135m", "360m"]), N=_log_int(rng, 1, 4096))


# ---------------------------------------------------------------- inputs

def _ld(c):
    return (c + 15) // 16 * 16


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 2654435761 % (1 << 62) + 97)
    return g


def _tokens(g, n, c):
    """Activations: each token of its own size, one channel in a hundred eight times as large as the others."""
    x = torch.randn(n, c, generator=g, device="cuda")
    gain = torch.where(torch.rand(c, generator=g, device="cuda") < 0.01, 8.0, 1.0)
    return x * gain * torch.exp(0.3 * torch.randn(n, 1, generator=g, device="cuda"))


def _coded(x):
    """Codes [rows][ld] and scales of a matrix that a user's program has quantized before."""
    top = x.abs().amax(dim=1)
    q = torch.round(x * (127 / top)[:, None])
    c = torch.zeros(x.shape[0], _ld(x.shape[1]), dtype=torch.int8, device="cuda")
    c[:, :x.shape[1]] = q.to(torch.int8)
    return c, top / 127


def _kind(name):
    return torch.bfloat16 if name == "bf16" else torch.float32


def _inputs(case, seed):
    """The inputs as plain tensors, a function of (case, seed)."""
    g, f = _gen(seed), case["family"]
    if f == "quantize":
        if case["src"] == "f32":  # weights
            return dict(x=torch.randn(case["M"], case["C"], generator=g, device="cuda") * 0.02)
        return dict(x=_tokens(g, case["M"], case["C"]).to(torch.bfloat16))
    if f == "norm":
        N, C = case["N"], case["C"]
        return dict(x=_tokens(g, N, C).to(_kind(case["src"])), r=_tokens(g, N, C),
                    w=1 + 0.1 * torch.randn(C, generator=g, device="cuda"))
    if f == "swiglu":  # f32: two matrices; bf16: one stacked product's halves
        N, H = case["N"], case["H"]
        if case["src"] == "f32":
            return dict(gate=_tokens(g, N, H), up=_tokens(g, N, H))
        gu = _tokens(g, N, 2 * H).to(torch.bfloat16)
        return dict(gu=gu, gate=gu[:, :H], up=gu[:, H:])
    if f == "matmul":
        a, sa = _coded(_tokens(g, case["M"], case["C"]))
        w, sw = _coded(torch.randn(case["OC"], case["C"], generator=g, device="cuda") * 0.02)
        return dict(a=a, sa=sa, w=w, sw=sw, C=case["C"],
                    b=torch.randn(case["OC"], generator=g, device="cuda") if case["bias"] else None)
    D, H = DIMS[case["model"]]
    w1, s1 = _coded(torch.randn(2 * H, D, generator=g, device="cuda") * 0.05)
    w2, s2 = _coded(torch.randn(D, H, generator=g, device="cuda") * 0.05)
    return dict(x=_tokens(g, case["N"], D).to(torch.bfloat16), r=_tokens(g, case["N"], D),
                w=1 + 0.1 * torch.randn(D, generator=g, device="cuda"), w1=w1, s1=s1, w2=w2, s2=s2, D=D, H=H)


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


_TYPES = {torch.float32: "<f4", torch.int8: "|i1", torch.bfloat16: "<i2"}


def _buffer(shape, dtype=torch.float32):
    """A backend buffer and a tensor over its memory."""
    n = math.prod(shape) * torch.empty(0, dtype=dtype).element_size()
    buf = _be().alloc(n)
    t = torch.as_tensor(_Shared(buf, shape, _TYPES[dtype]), device="cuda")
    return buf, t.view(dtype)


def _upload(values):
    """A backend buffer holding a tensor's values (the buffer's zero fill is over first)."""
    buf, t = _buffer(values.shape, values.dtype)
    _be().synchronize()
    t.copy_(values)
    return buf


def _i32(*v):
    return _be().params(*v)


class _Encoded:
    """The dispatches of one pass, bound once; each call encodes and commits them, and takes back the encoder of its
    previous call, so that a program keeps the GPU busy."""

    def __init__(self, calls):
        import bmhip
        be = _be()
        self.lib, self.keep, self.args, self.enc = bmhip.lib(), calls, [], None
        for name, bufs, grid, offsets in calls:
            n = len(bufs)
            arr = (ctypes.c_void_p * n)(*[b.h for b in bufs])
            off = (ctypes.c_size_t * n)(*offsets) if offsets else None
            self.args.append((be.kernel(name).h, arr, off, n, grid[0], grid[1] if len(grid) > 1 else 1, 1, 256, 1, 1))

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


def _suffix(kind):
    return "_bf16" if kind in ("bf16", torch.bfloat16) else ""


def _bind(case, i):
    """The pass's dispatches over backend buffers, and its outputs."""
    f = case["family"]
    if f == "quantize":
        M, C = case["M"], case["C"]
        src, q = _upload(i["x"]), _buffer((M, _ld(C)), torch.int8)[0]
        (s, st), (v, vt) = _buffer((M,)), _buffer((M, C), torch.bfloat16)
        return _Encoded([
            ("quantize_rows_i8" + _suffix(case["src"]), [src, q, s, _i32(M, C, C, _ld(C))], (M,), None),
            ("dequantize_rows_i8_bf16", [q, s, v, _i32(M, C, _ld(C), C)], (M,), None),
        ]), dict(scale=st, values=vt)
    if f == "norm":
        N, C = case["N"], case["C"]
        x, r, w = _upload(i["x"]), _upload(i["r"]), _upload(i["w"])
        q = _buffer((N, _ld(C)), torch.int8)[0]
        (h, ht), (s, st), (v, vt) = _buffer((N, C)), _buffer((N,)), _buffer((N, C), torch.bfloat16)
        return _Encoded([
            ("rmsnorm_forward_i8" + _suffix(case["src"]),
             [x, r, w, h, q, s, _i32(N, C, _ld(C), 1), _be().upload(np.float32([EPS]))], (N,), None),
            ("dequantize_rows_i8_bf16", [q, s, v, _i32(N, C, _ld(C), C)], (N,), None),
        ]), dict(h=ht, scale=st, values=vt)
    if f == "swiglu":
        N, H = case["N"], case["H"]
        if case["src"] == "f32":
            gate, up, ld, offsets = _upload(i["gate"]), _upload(i["up"]), H, None
        else:
            gate = up = _upload(i["gu"])
            ld, offsets = 2 * H, [0, 2 * H, 0, 0, 0]
        q = _buffer((N, _ld(H)), torch.int8)[0]
        (s, st), (v, vt) = _buffer((N,)), _buffer((N, H), torch.bfloat16)
        return _Encoded([
            ("swiglu_forward_i8" + _suffix(case["src"]), [gate, up, q, s, _i32(N, H, ld, _ld(H))], (N,), offsets),
            ("dequantize_rows_i8_bf16", [q, s, v, _i32(N, H, _ld(H), H)], (N,), None),
        ]), dict(scale=st, values=vt)
    if f == "matmul":
        M, C, OC, kind = case["M"], case["C"], case["OC"], _kind(case["out"])
        a, sa, w, sw = (_upload(i[k]) for k in ("a", "sa", "w", "sw"))
        b = _upload(i["b"]) if case["bias"] else sw
        o, ot = _buffer((M, OC), kind)
        return _Encoded([("matmul_forward_i8" + _suffix(kind), [a, sa, w, sw, b, o, _i32(
            M, C, OC, int(case["bias"]), _ld(C), _ld(C), OC)], (OC, M), None)]), dict(out=ot)
    N, D, H, B = case["N"], i["D"], i["H"], torch.bfloat16
    x, r, w, w1, s1, w2, s2 = (_upload(i[k]) for k in ("x", "r", "w", "w1", "s1", "w2", "s2"))
    q1, q2 = _buffer((N, _ld(D)), torch.int8)[0], _buffer((N, _ld(H)), torch.int8)[0]
    c1, c2, gu = _buffer((N,))[0], _buffer((N,))[0], _buffer((N, 2 * H), B)[0]
    (h, ht), (y, yt) = _buffer((N, D)), _buffer((N, D), B)
    return _Encoded([
        ("rmsnorm_forward_i8_bf16", [x, r, w, h, q1, c1, _i32(N, D, _ld(D), 1), _be().upload(np.float32([EPS]))], (N,),
         None),
        ("matmul_forward_i8_bf16", [q1, c1, w1, s1, s1, gu, _i32(N, D, 2 * H, 0, _ld(D), _ld(D), 2 * H)], (2 * H, N),
         None),
        ("swiglu_forward_i8_bf16", [gu, gu, q2, c2, _i32(N, H, 2 * H, _ld(H))], (N,), [0, 2 * H, 0, 0, 0]),
        ("matmul_forward_i8_bf16", [q2, c2, w2, s2, s2, y, _i32(N, H, D, 0, _ld(H), _ld(H), D)], (D, N), None),
    ]), dict(h=ht, y=yt)


def prepare(case, seed):
    i = _inputs(case, seed)
    if own:  # the framework's kernels take the backend's own buffers
        call, out = _bind(case, i)
        torch.cuda.synchronize()
        return dict(call=call, out=out)
    return dict(i, family=case["family"], kind=_kind(case.get("out", "bf16")))


# ---------------------------------------------------------------- the plain forms

def _codes(p):
    """Codes of each row, whole numbers in fp32, and the row's largest magnitude."""
    top = p.abs().amax(dim=1)
    inv = 127 / top
    inv = torch.where(torch.isfinite(inv), inv, torch.zeros_like(inv))
    return torch.round(p * inv[:, None]).clamp(-127, 127), top


def _norm(x, r, w):
    h = x.float() + r
    q, top = _codes(h * w)
    scale = top.double() / torch.sqrt(h.double().square().mean(dim=1) + EPS) / 127
    return h, q, scale.float()


def _swiglu(gate, up):
    g = gate.float()
    q, top = _codes(g / (1 + torch.exp(-g)) * up.float())
    return q, top / 127


def _product(q, sa, w, sw, C, b, kind):
    y = q[:, :C].float() @ w[:, :C].float().T * sa[:, None] * sw
    return (y if b is None else y + b).to(kind)


def _values(q, scale):
    return (q * scale[:, None]).to(torch.bfloat16)


def run(s):
    if own:
        s["call"]()
        return s["out"]
    f = s["family"]
    if f == "quantize":
        q, top = _codes(s["x"].float())
        return dict(scale=top / 127, values=_values(q, top / 127))
    if f == "norm":
        h, q, scale = _norm(s["x"], s["r"], s["w"])
        return dict(h=h, scale=scale, values=_values(q, scale))
    if f == "swiglu":
        q, scale = _swiglu(s["gate"], s["up"])
        return dict(scale=scale, values=_values(q, scale))
    if f == "matmul":
        return dict(out=_product(s["a"], s["sa"], s["w"], s["sw"], s["C"], s["b"], s["kind"]))
    H = s["H"]
    h, q, scale = _norm(s["x"], s["r"], s["w"])
    gu = _product(q, scale, s["w1"], s["s1"], s["D"], None, torch.bfloat16)
    q, scale = _swiglu(gu[:, :H], gu[:, H:])
    return dict(h=h, y=_product(q, scale, s["w2"], s["s2"], H, None, torch.bfloat16))


# ---------------------------------------------------------------- work

def work(case):
    f = case["family"]
    n = 2 if case.get("src") == "bf16" else 4
    if f == "quantize":  # source; codes, scales and values
        M, C = case["M"], case["C"]
        return dict(bytes=M * C * (n + 1 + 2) + 4 * M, flops=4 * M * C)
    if f == "norm":  # branch, residual and gains; sum, codes, scales and values
        N, C = case["N"], case["C"]
        return dict(bytes=N * C * (n + 4 + 4 + 1 + 2) + 4 * (N + C), flops=8 * N * C)
    if f == "swiglu":
        N, H = case["N"], case["H"]
        return dict(bytes=N * H * (2 * n + 1 + 2) + 4 * N, flops=9 * N * H)
    if f == "matmul":
        M, C, OC = case["M"], case["C"], case["OC"]
        return dict(bytes=(M + OC) * (C + 4) + 4 * OC * case["bias"] + M * OC * (2 if case["out"] == "bf16" else 4),
                    flops=2 * M * C * OC)
    (D, H), N = DIMS[case["model"]], case["N"]  # what enters and leaves the MLP, and its weights
    return dict(bytes=3 * D * H + 4 * (2 * H + 2 * D) + N * D * (2 + 4 + 4 + 2), flops=6 * N * D * H)


# ---------------------------------------------------------------- the same in 64 bits

def _round_rows(p):
    """Nearest code of each value of a row on the grid of its largest magnitude, and the grid's step, in 64 bits."""
    step = p.abs().max(dim=1, keepdim=True).values / 127
    return torch.where(step > 0, torch.round(p / torch.where(step > 0, step, torch.ones_like(step))), 0.0), step


def exact(case, seed):
    i, f = _inputs(case, seed), case["family"]
    d = {k: v.double() for k, v in i.items() if isinstance(v, torch.Tensor)}
    if f == "quantize":
        c, step = _round_rows(d["x"])
        return dict(scale=step[:, 0], values=c * step)
    if f == "swiglu":
        c, step = _round_rows(d["gate"] * torch.sigmoid(d["gate"]) * d["up"])
        return dict(scale=step[:, 0], values=c * step)
    if f == "matmul":
        C = case["C"]
        y = (d["a"][:, :C] * d["sa"][:, None]) @ (d["w"][:, :C] * d["sw"][:, None]).T
        return dict(out=y + d["b"] if case["bias"] else y)
    h = (i["x"].float() + i["r"]).double()  # the residual stream is kept in fp32
    rms = torch.sqrt((h * h).sum(dim=1, keepdim=True) / h.shape[1] + EPS)
    c, step = _round_rows(h / rms * d["w"])
    if f == "norm":
        return dict(h=h, scale=step[:, 0], values=c * step)
    D, H = i["D"], i["H"]
    gu = ((c * step) @ (d["w1"][:, :D] * d["s1"][:, None]).T).to(torch.bfloat16).double()
    c, step = _round_rows(gu[:, :H] * torch.sigmoid(gu[:, :H]) * gu[:, H:])
    return dict(h=h, y=(c * step) @ (d["w2"][:, :H] * d["s2"][:, None]).T)
