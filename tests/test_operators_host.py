"""What the operators on device tensors refuse, before any device work: no GPU needed."""
import ctypes

import pytest

import hat_amd as hl


class Fake:
    """A tensor of device 0 in everything but memory."""

    def __init__(self, *shape, dtype="float32", strides=None, ptr=1 << 20, device=0):
        self.shape, self.dtype, self.ptr, self.device = shape, dtype, ptr, device
        s, out = 1, []
        for n in reversed(shape):
            out.append(s)
            s *= n
        self.strides = strides or tuple(reversed(out))

    def data_ptr(self):
        return self.ptr

    def get_device(self):
        return self.device

    def stride(self):
        return self.strides


def refused(needle, f, *a, **kw):
    with pytest.raises(hl.HatError) as e:
        f(*a, **kw)
    assert needle in str(e.value), str(e.value)


def i32(*shape, **kw):
    return Fake(*shape, dtype="int32", **kw)


Q, K, POS = Fake(2, 5, 4, 32), Fake(2, 5, 2, 32), i32(5, 2)


@pytest.mark.parametrize("needle,args,kw", [
    ("do not fit a head_dim", (Q, K, POS, [9, 8]), {}),
    ("do not fit a head_dim", (Q, K, POS, [0, 0]), {}),
    ("section -1", (Q, K, POS, [-1, 8]), {}),
    ("2 axes of positions and 1 sections", (Q, K, POS, [8]), {}),
    ("int32 expected", (Q, K, Fake(5, 2), [4, 4]), {}),
    ("is no [5, axis]", (Q, K, i32(6, 2), [4, 4]), {}),
    ("does not go with q", (Q, Fake(2, 6, 2, 32), POS, [4, 4]), {}),
    ("differs from the first", (Q, Fake(2, 5, 2, 32, dtype="float16"), POS, [4, 4]), {}),
    ("type torch.int64", (Fake(2, 5, 4, 32, dtype="torch.int64"), None, POS, [4, 4]), {}),
    ("type 3", (i32(2, 5, 4, 32), None, POS, [4, 4]), {}),
    ("not a tensor of device 0", (Fake(2, 5, 4, 32, device=-1), None, POS, [4, 4]), {}),
    ("not a tensor of device 0", (Fake(2, 5, 4, 32, device=1), None, POS, [4, 4]), {}),
    ("stride 1", (Fake(2, 5, 4, 32, strides=(1280, 256, 64, 2)), None, POS, [4, 4]), {}),
    ("head_dim 258", (Fake(1, 5, 1, 258), None, POS, [4, 4]), {}),
    ("base must be positive", (Q, K, POS, [4, 4]), dict(base=0.0)),
    ("base must be positive", (Q, K, POS, [4, 4]), dict(base=float("nan"))),
    ("halves or neighbours", (Q, K, POS, [4, 4]), dict(pairs="thirds")),
    ("k_out without k", (Q, None, POS, [4, 4]), dict(k_out=K)),
    ("is expected", (Q, K, POS, [4, 4]), dict(q_out=K)),
    ("other strides", (Q, None, POS, [4, 4]), dict(q_out=Fake(2, 5, 4, 32, strides=(1280, 256, 64, 1)))),
    ("on top of one another", (Q, None, POS, [4, 4]), dict(q_out=Fake(2, 5, 4, 32, strides=(0, 128, 32, 1), ptr=1 << 22))),
    ("not aligned", (Fake(2, 5, 4, 32, ptr=(1 << 20) + 2), None, POS, [4, 4]), {}),
    ("has a stride of -128", (Fake(2, 5, 4, 32, strides=(640, -128, 32, 1)), None, POS, [4, 4]), {}),
    ("null", (Fake(2, 5, 4, 32, ptr=0), None, POS, [4, 4]), {}),
])
def test_rotary_refuses(needle, args, kw):
    refused(needle, hl.op_rotary, *args, **kw)


V, OUT = Fake(2, 5, 2, 32), Fake(2, 5, 4, 32, ptr=1 << 24)
PQ, PK, PO = Fake(9, 4, 32), Fake(9, 2, 32), Fake(9, 4, 32, ptr=1 << 24)


@pytest.mark.parametrize("needle,args,kw", [
    ("do not divide", (Fake(2, 5, 5, 32), K, V, Fake(2, 5, 5, 32, ptr=1 << 24)), {}),
    ("head_dim 129", (Fake(1, 5, 1, 129), Fake(1, 5, 1, 129), Fake(1, 5, 1, 129), Fake(1, 5, 1, 129, ptr=1 << 24)), {}),
    ("head_dim 32 of q and 16 of k", (Q, Fake(2, 5, 2, 16), Fake(2, 5, 2, 16), OUT), {}),
    ("is expected", (Q, K, Fake(2, 6, 2, 32), OUT), {}),
    ("is expected", (Q, K, V, Fake(2, 5, 2, 32)), {}),
    ("are not 2 sequences", (Q, Fake(3, 5, 2, 32), Fake(3, 5, 2, 32), OUT), {}),
    ("differs from the first", (Q, Fake(2, 5, 2, 32, dtype="bfloat16"), V, OUT), {}),
    ("scale must be finite", (Q, K, V, OUT), dict(scale=float("inf"))),
    ("cap must be 0 or positive", (Q, K, V, OUT), dict(cap=-1.0)),
    ("cap must be 0 or positive", (Q, K, V, OUT), dict(cap=float("nan"))),
    ("next to nothing", (Q, K, V, OUT), dict(cap=1e-9)),
    ("next to nothing", (Q, K, V, OUT), dict(cap=1e-3, scale=2000.0)),
    ("belongs to the causal mask", (Q, K, V, OUT), dict(prefix=i32(2))),
    ("2 contiguous values of int32", (Q, K, V, OUT), dict(prefix=i32(3), causal=True)),
    ("2 contiguous values of int32", (Q, K, V, OUT), dict(k_lens=Fake(2))),
    ("4 contiguous values of fp32", (Q, K, V, OUT), dict(slopes=Fake(2))),
    ("go together", (Q, K, V, OUT), dict(slopes=Fake(4), pos_q=POS)),
    ("positions without slopes", (Q, K, V, OUT), dict(pos_q=POS, pos_k=POS)),
    ("axes 5", (Q, K, V, OUT), dict(slopes=Fake(4), pos_q=i32(5, 5), pos_k=i32(5, 5))),
    ("2 axes in pos_q and 1", (Q, K, V, OUT), dict(slopes=Fake(4), pos_q=POS, pos_k=i32(5, 1))),
    ("offsets, not lengths", (PQ, PK, PK, PO), dict(cu_q=i32(4), cu_k=i32(4), k_lens=i32(3))),
    ("3 sequences in cu_q and 2 in cu_k", (PQ, PK, PK, PO), dict(cu_q=i32(4), cu_k=i32(3))),
    ("a packed tensor is", (Q, K, V, OUT), dict(cu_q=i32(3), cu_k=i32(3))),
    ("are not 3 sequences", (PQ, PK, PK, PO), dict(cu_q=i32(4))),
    ("offsets of every sequence", (PQ, PK, PK, PO), dict(cu_q=i32(0), cu_k=i32(0))),
    ("out overlaps", (Q, K, V, Fake(2, 5, 4, 32, strides=(1280, 256, 64, 1))), {}),
    ("on top of one another", (Q, K, V, Fake(2, 5, 4, 32, strides=(640, 128, 0, 1), ptr=1 << 24)), {}),
    ("token stride 4194304", (Q, Fake(2, 5, 2, 32, strides=(1 << 25, 1 << 22, 32, 1)), V, OUT), {}),
    ("one contiguous row", (Q, K, V, OUT), dict(workspace=Fake(2, 2, dtype="uint8"))),
    ("not a tensor of device 0", (Q, K, V, OUT), dict(workspace=Fake(2, dtype="uint8", device=-1))),
])
def test_attention_refuses(needle, args, kw):
    refused(needle, hl.op_attention, *args, **kw)


X, Y, XO, H = Fake(6, 144), Fake(6, 144), Fake(6, 144, ptr=1 << 23), Fake(6, 144, ptr=1 << 24)


@pytest.mark.parametrize("needle,args,kw", [
    ("no output", (X, Y), {}),
    ("width 16385", (Fake(1, 16385), None, None, Fake(1, 16385)), {}),
    ("type int32", (i32(6, 144), None, None, i32(6, 144)), {}),
    ("is no [rows, width]", (X, Fake(6, 143), XO, H), {}),
    ("is no [rows, width]", (Fake(6, 144, strides=(288, 2)), None, None, H), {}),
    ("differs from x's", (X, Fake(6, 144, dtype="float16"), XO, H), {}),
    ("gates of (4, 144)", (X, Y, XO, H), dict(gate=Fake(4, 144))),
    ("gates of (1, 9)", (X, Y, XO, H), dict(gate=Fake(1, 9))),
    ("a norm or a gate of no y", (X, None, XO, H), dict(gate=Fake(1, 144))),
    ("a norm or a gate of no y", (X, None, XO, H), dict(post="rms")),
    ("weights of no norm", (X, Y, XO, H), dict(post_weight=Fake(144))),
    ("weights of no norm", (X, Y, XO, H), dict(pre_bias=Fake(144))),
    ("144 contiguous values of fp32", (X, Y, XO, H), dict(pre="rms", pre_weight=Fake(144, dtype="float16"))),
    ("none, layer or rms", (X, Y, XO, H), dict(pre="batch")),
    ("eps 0 or positive", (X, Y, XO, H), dict(pre="rms", eps=-1.0)),
    ("scale must be finite", (X, Y, XO, H), dict(scale=float("nan"))),
    ("the same rows", (X, Y, XO, XO), {}),
    ("other strides", (X, Y, Fake(6, 144, strides=(160, 1)), H), {}),
    ("on top of one another", (X, Y, Fake(6, 144, strides=(100, 1), ptr=1 << 23), H), {}),
    ("not a tensor of device 0", (X, Y, XO, Fake(6, 144, device=-1)), {}),
])
def test_residual_norm_refuses(needle, args, kw):
    refused(needle, hl.op_residual_norm, *args, **kw)


def test_c_entries_refuse_null_and_unknown_types():
    L = hl.lib()
    assert L.hat_op_rotary(None, None) == -1 and "null" in hl._err()
    assert L.hat_op_attention(None, None) == -1 and "null" in hl._err()
    assert L.hat_op_residual_norm(None, None) == -1 and "null" in hl._err()
    assert L.hat_op_attention_workspace(None) == ctypes.c_size_t(-1).value and "null" in hl._err()
    a = hl.ResidualNormArgs()
    a.dtype = 7
    assert L.hat_op_residual_norm(ctypes.byref(a), None) == -1 and "type 7" in hl._err()
    b = hl.AttentionArgs()
    b.q_heads, b.kv_heads, b.head_dim, b.n_seq, b.q_tokens, b.k_tokens = 4, 2, 32, 1, 1 << 33, 8
    assert L.hat_op_attention(ctypes.byref(b), None) == -1 and "q_tokens" in hl._err()


def test_structures_are_the_header_s():
    """The binding's structures against the header's, compiled."""
    import os
    import subprocess
    import tempfile
    names = {"hat_rotary": hl.RotaryArgs, "hat_attention": hl.AttentionArgs, "hat_residual_norm": hl.ResidualNormArgs,
             "hat_heads": hl.Heads, "hat_positions": hl.Positions}
    src = '#include <stdio.h>\n#include <stddef.h>\n#include "hat.h"\nint main(void){\n'
    for c, t in names.items():
        src += f'printf("%zu\\n", sizeof({c}));\n'
        for f in t._fields_:
            src += f'printf("%zu\\n", offsetof({c}, {f[0]}));\n'
    with tempfile.TemporaryDirectory() as d:
        with open(os.path.join(d, "a.c"), "w") as f:
            f.write(src + "return 0;}\n")
        exe = os.path.join(d, "a")
        subprocess.run(["gcc", "-I", os.path.dirname(hl.HEADER), "-o", exe, os.path.join(d, "a.c")], check=True)
        got = [int(x) for x in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for t in names.values():
        want += [ctypes.sizeof(t)] + [getattr(t, f[0]).offset for f in t._fields_]
    assert got == want


def test_packed_layouts_are_the_structures():
    """The layouts that calls pack against the structures of the same fields."""
    def leaves(t, path=()):
        for name, kind in t._fields_:
            if hasattr(kind, "_fields_"):
                yield from leaves(kind, path + (name,))
            elif hasattr(kind, "_length_"):
                yield from ((path + (name, i), kind._type_) for i in range(kind._length_))
            else:
                yield path + (name,), kind

    for layout, t in ((hl._ROTARY, hl.RotaryArgs), (hl._ATTENTION, hl.AttentionArgs), (hl._NORM, hl.ResidualNormArgs)):
        a, values = t(), []
        for n, (path, kind) in enumerate(leaves(t), 1):
            to = a
            for step in path[:-1]:
                to = getattr(to, step) if isinstance(step, str) else to[step]
            if isinstance(path[-1], str):
                setattr(to, path[-1], n)
            else:
                to[path[-1]] = n
            values.append(n)
        if t is hl.AttentionArgs:  # the gap between cap and slopes is a field of the layout
            values.insert(values.index([i for i, (p, _) in enumerate(leaves(t), 1) if p == ("slopes",)][0]), 0.0)
        assert layout.pack(*values) == bytes(a)
