"""The context layer's and the optimizer's entry points on the host (CPU only, no kernel launches): argument structs as
the header has them, and what is refused before any launch, in C and in Python."""
from __future__ import annotations

import ctypes
import subprocess

import pytest
import torch

from rsna_knee_efficiency_amd import context, hip, optim

P = 1 << 20                                    # a pointer that no refused call follows


def test_struct_layouts_match_header(tmp_path):
    pairs = [("D8sNormArgs", hip.NormArgs, ("partial_bytes", "rows", "width", "eps")),
             ("D8sRotaryArgs", hip.RotaryArgs, ("pos", "pos_ss", "B", "inverse", "freq", "axis")),
             ("D8sAttnArgs", hip.AttnArgs, ("mask", "workspace", "q_sb", "mask_sb", "B", "sinks", "scale")),
             ("D8sTokenArgs", hip.TokenArgs, ("lengths", "v_sh", "B", "sinks", "scale")),
             ("D8sAdamwTensor", hip.AdamwTensor, ("g", "n", "at")),
             ("D8sAdamwArgs", hip.AdamwArgs, ("grad_scale", "step", "lr", "weight_decay", "count", "bits"))]
    lines = "".join(f'  printf("%zu {" ".join(["%zu"] * len(f))}\\n", sizeof({c}), '
                    + ", ".join(f"offsetof({c}, {n})" for n in f) + ");\n" for c, _, f in pairs)
    prog = tmp_path / "layout.c"
    prog.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "d8s_hip.h"\nint main(void) {\n' + lines
                    + '  printf("%d %d %d\\n", D8S_ROTARY_PAIRS, D8S_ADAMW_BLOCK, D8S_F16);\n  return 0; }\n')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", f"-I{hip.HEADER.parent}", str(prog), "-o", str(exe)], check=True)
    got = [list(map(int, x.split())) for x in
           subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines()]
    for (_, s, fields), row in zip(pairs, got):
        assert row == [ctypes.sizeof(s), *(getattr(s, n).offset for n in fields)], s
    assert got[-1] == [hip.ROTARY_PAIRS, hip.ADAMW_BLOCK, hip.ELEMENTS[torch.float16]]
    assert optim._ROW.itemsize == ctypes.sizeof(hip.AdamwTensor)


def _norm(**kw):
    a = hip.NormArgs(x=P, w=P, b=P, y=P, dy=P, dx=P, dw=P, db=P, mean=P, rstd=P, partial=P, partial_bytes=1 << 40,
                     rows=4, x_stride=64, dy_stride=64, width=64, eps=1e-5)
    for k, v in kw.items():
        setattr(a, k, v)
    return ctypes.byref(a)


def _rotary(axis=0, **kw):
    a = hip.RotaryArgs(x=P, y=P, pos=P, B=1, S=4, H=2, D=64, pairs=32, axes=3, dtype=1)
    a.axis[5] = axis
    for k, v in kw.items():
        setattr(a, k, v)
    return ctypes.byref(a)


def _attn(**kw):
    a = hip.AttnArgs(**{n: P for n in ("q", "k", "v", "out", "lse", "dout", "dq", "dk", "dv", "workspace")},
                     ws_bytes=1 << 40, B=2, S=100, H=4, HK=2, D=64, dtype=1, left=10, right=0, sinks=2, scale=0.125)
    for k, v in kw.items():
        setattr(a, k, v)
    return ctypes.byref(a)


def _token(**kw):
    a = hip.TokenArgs(**{n: P for n in ("q", "k", "v", "lengths", "out", "workspace")}, ws_bytes=1 << 40, B=2, S=1000,
                      H=4, HK=2, D=64, dtype=1, left=500, sinks=2, scale=0.125)
    for k, v in kw.items():
        setattr(a, k, v)
    return ctypes.byref(a)


_TENSORS = (hip.AdamwTensor * 2)(hip.AdamwTensor(P, P, 300, 0), hip.AdamwTensor(P, P, 5, 512))


def _adamw(at=512, g=P, **kw):
    rows = (hip.AdamwTensor * 2)(hip.AdamwTensor(P, P, 300, 0), hip.AdamwTensor(P, g, 5, at))
    a = hip.AdamwArgs(tensors=ctypes.addressof(rows), m=P, v=P, m_scale=P, v_scale=P, step=1, lr=1e-3, beta1=0.9,
                      beta2=0.999, eps=1e-8, count=2, dtype=0, grad_dtype=0, bits=32)
    a.kept = rows
    for k, v in kw.items():
        setattr(a, k, v)
    return ctypes.byref(a)


@pytest.mark.parametrize("name,args", [
    ("d8s_layer_norm", lambda: (None, None)),
    ("d8s_layer_norm", lambda: (_norm(dtype=3), None)),
    ("d8s_layer_norm", lambda: (_norm(dtype=1, wdtype=2), None)),
    ("d8s_layer_norm", lambda: (_norm(width=0), None)),
    ("d8s_layer_norm", lambda: (_norm(width=16385, x_stride=16385), None)),
    ("d8s_layer_norm", lambda: (_norm(rows=0), None)),
    ("d8s_layer_norm", lambda: (_norm(x_stride=63), None)),
    ("d8s_layer_norm", lambda: (_norm(y=0), None)),
    ("d8s_layer_norm", lambda: (_norm(mean=0), None)),
    ("d8s_layer_norm_workspace", lambda: (_norm(), None)),
    ("d8s_layer_norm_backward", lambda: (_norm(partial_bytes=64 * 8 - 1), None)),
    ("d8s_layer_norm_backward", lambda: (_norm(dy_stride=10), None)),
    ("d8s_layer_norm_backward", lambda: (_norm(dw=0), None)),
    ("d8s_rotary", lambda: (None, None)),
    ("d8s_rotary", lambda: (_rotary(pairs=33), None)),
    ("d8s_rotary", lambda: (_rotary(pairs=0), None)),
    ("d8s_rotary", lambda: (_rotary(D=1024, pairs=257), None)),
    ("d8s_rotary", lambda: (_rotary(axis=3), None)),
    ("d8s_rotary", lambda: (_rotary(pos_type=3), None)),
    ("d8s_rotary", lambda: (_rotary(B=1 << 20, S=1 << 20), None)),
    ("d8s_attention", lambda: (None, None)),
    ("d8s_attention", lambda: (_attn(dtype=0), None)),
    ("d8s_attention", lambda: (_attn(D=96), None)),
    ("d8s_attention", lambda: (_attn(H=5), None)),
    ("d8s_attention", lambda: (_attn(HK=0), None)),
    ("d8s_attention", lambda: (_attn(S=0), None)),
    ("d8s_attention", lambda: (_attn(left=-1), None)),
    ("d8s_attention", lambda: (_attn(sinks=-1), None)),
    ("d8s_attention", lambda: (_attn(scale=0.0), None)),
    ("d8s_attention", lambda: (_attn(scale=float("inf")), None)),
    ("d8s_attention", lambda: (_attn(scale=float("nan")), None)),
    ("d8s_attention", lambda: (_attn(q=0), None)),
    ("d8s_attention", lambda: (_attn(B=1 << 12, S=1 << 20), None)),
    ("d8s_attention_workspace", lambda: (_attn(), None)),
    ("d8s_attention_backward", lambda: (_attn(ws_bytes=100), None)),
    ("d8s_attention_backward", lambda: (_attn(workspace=P + 8), None)),
    ("d8s_attention_backward", lambda: (_attn(lse=0), None)),
    ("d8s_attention_token", lambda: (_token(lengths=0), None)),
    ("d8s_attention_token", lambda: (_token(ws_bytes=0), None)),
    ("d8s_attention_token", lambda: (_token(D=32), None)),
    ("d8s_attention_token", lambda: (_token(left=-1), None)),
    ("d8s_attention_token", lambda: (_token(H=3), None)),
    ("d8s_adamw", lambda: (None, None)),
    ("d8s_adamw", lambda: (_adamw(bits=16), None)),
    ("d8s_adamw", lambda: (_adamw(dtype=1, grad_dtype=2), None)),
    ("d8s_adamw", lambda: (_adamw(count=0), None)),
    ("d8s_adamw", lambda: (_adamw(at=500), None)),
    ("d8s_adamw", lambda: (_adamw(g=0), None)),
    ("d8s_adamw", lambda: (_adamw(step=0), None)),
    ("d8s_adamw", lambda: (_adamw(beta2=1.0), None)),
    ("d8s_adamw", lambda: (_adamw(bits=8, m_scale=0), None)),
    ("d8s_adamw", lambda: (_adamw(m=P + 1), None)),
    ("d8s_adamw_moments", lambda: (P, P, P, P, 255, P, P, None)),
    ("d8s_adamw_moments", lambda: (P, P, P, 0, 256, P, P, None)),
])
def test_invalid_arguments_fail_on_the_host(name, args):
    with pytest.raises(hip.D8sError, match=name):
        hip.call(name, *args())


def _t(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


BF = torch.bfloat16


@pytest.mark.parametrize("call,match", [
    (lambda: context.layer_norm(_t(4, 8), _t(8)), "one GPU"),
    (lambda: context.layer_norm(_t(4, 8), _t(7)), "weight"),
    (lambda: context.layer_norm(_t(4, 8), _t(8), _t(8, dtype=BF)), "bias"),
    (lambda: context.layer_norm(_t(4, 8, dtype=BF), _t(8, dtype=torch.float16)), "weight"),
    (lambda: context.layer_norm(_t(4, 8, dtype=torch.float64), _t(8)), "float32"),
    (lambda: context.layer_norm(_t(1, 16385), _t(16385)), "16384"),
    (lambda: context.layer_norm(_t(1, 0), _t(0)), "16384"),
    (lambda: context.layer_norm_backward(_t(4, 7), _t(4, 8), _t(8), _t(4), _t(4)), "dy"),
    (lambda: context.layer_norm_backward(_t(4, 8), _t(4, 8), _t(8), _t(5), _t(4)), "mean"),
    (lambda: context.rotary(_t(1, 4, 2, 16), _t(4, 3, dtype=torch.int32), (3, 3, 3)), "channels"),
    (lambda: context.rotary(_t(1, 4, 2, 16), _t(4, 2, dtype=torch.int32), (3, 3, 2)), "positions"),
    (lambda: context.rotary(_t(1, 4, 2, 16), _t(4, 1, dtype=torch.int16), (8,)), "positions"),
    (lambda: context.rotary(_t(1, 4, 2, 16), _t(4, 1, dtype=torch.int32), (8,)), "one GPU"),
    (lambda: context.rotary(_t(1, 4, 2, 16), _t(4, 1, dtype=torch.int32), ()), "sections"),
    (lambda: context.rotary(_t(1, 4, 2, 16), _t(4, 1, dtype=torch.int32), (8,), base=0.0), "base"),
    (lambda: context.rotary(_t(4, 2, 16), _t(4, 1, dtype=torch.int32), (8,)), "x must be"),
    (lambda: context.window_attention(*(_t(1, 4, 2, 64) for _ in range(3))), "bfloat16"),
    (lambda: context.window_attention(*(_t(1, 4, 2, 32, dtype=BF) for _ in range(3))), "64 or 128"),
    (lambda: context.window_attention(*(_t(1, 4, 2, 64, dtype=BF) for _ in range(3))), "one GPU"),
    (lambda: context.window_attention(_t(1, 4, 3, 64, dtype=BF), *(_t(1, 4, 2, 64, dtype=BF) for _ in range(2))), "divide"),
    (lambda: context.window_attention(_t(1, 4, 2, 64, dtype=BF), *(_t(1, 5, 2, 64, dtype=BF) for _ in range(2))), "tokens"),
    (lambda: context.window_attention(*(_t(1, 4, 2, 64, dtype=BF) for _ in range(3)), scale=-1.0), "scale"),
    (lambda: context.window_attention_token(_t(1, 2, 64, dtype=BF), *(_t(1, 9, 2, 64, dtype=BF) for _ in range(2)),
                                            _t(1, dtype=torch.int64)), "lengths"),
    (lambda: context.window_attention_token(_t(1, 2, 64, dtype=BF), *(_t(1, 9, 3, 64, dtype=BF) for _ in range(2)),
                                            _t(1, dtype=torch.int32)), "divide"),
    (lambda: optim.AdamW([]), "no parameters"),
    (lambda: optim.AdamW([_t(3)]), "one GPU"),
    (lambda: optim.AdamW([_t(3)], state_bits=4), "state_bits"),
    (lambda: optim.AdamW([_t(3)] * 2), "twice"),
    (lambda: optim.AdamW([_t(3)], betas=(0.9, 1.0)), "betas"),
])
def test_python_refuses(call, match):
    with pytest.raises(ValueError, match=match):
        call()


def test_workspaces_follow_the_sizes():
    need = ctypes.c_uint64()

    def of(name, args):
        hip.call(name, args, ctypes.byref(need))
        return need.value
    assert of("d8s_layer_norm_workspace", _norm(rows=1)) == 2 * 64 * 4
    assert of("d8s_layer_norm_workspace", _norm(rows=1 << 30)) == of("d8s_layer_norm_workspace", _norm(rows=1 << 29))
    # one float32 a query and head, and none more where no tile of keys is split
    assert of("d8s_attention_workspace", _attn(B=64, S=1024, H=16, HK=16, sinks=0)) == 64 * 16 * 1024 * 4
    assert of("d8s_attention_workspace", _attn(B=64, S=1024, H=16, HK=16, sinks=1)) > 64 * 16 * 1024 * 4
    assert of("d8s_attention_token_workspace", _token(S=100)) == 0
    assert of("d8s_attention_token_workspace", _token()) % (2 * 4 * (64 + 2) * 4) == 0
