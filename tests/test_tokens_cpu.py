"""What the embedding and vocabulary operators refuse, before any launch: arguments through the
package's entry points, and args structs through the C ABI."""

import ctypes

import pytest
import torch


def test_embedding_refuses_bad_arguments(m3):
    K, table, tokens = m3.kernels, torch.zeros(5, 4), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="ROCm device only"):
        m3.embed_tokens(table, tokens)
    with pytest.raises(ValueError, match="int32 or int64"):
        m3.embed_tokens(table, tokens.float())
    with pytest.raises(ValueError, match="bf16 or f32"):
        m3.embed_tokens(table.double(), tokens)
    with pytest.raises(ValueError, match="must be \\(V, D\\)"):
        m3.embed_tokens(table[0], tokens)
    with pytest.raises(ValueError, match="must not be empty"):
        m3.embed_tokens(table[:0], tokens)
    for pad in (5, -6):
        with pytest.raises(ValueError, match="padding_idx"):
            m3.embed_tokens(table, tokens, padding_idx=pad)
        with pytest.raises(ValueError, match="padding_idx"):
            K.embedding_backward(tokens, torch.zeros(3, 4), 5, padding_idx=pad)
    with pytest.raises(ValueError, match="tokens.shape"):
        K.embedding_backward(tokens, torch.zeros(2, 4), 5)
    with pytest.raises(ValueError, match="must not be empty"):
        K.embedding_backward(tokens, torch.zeros(3, 4), 0)


def test_embed_abi_refuses_bad_structs(m3):
    from mamba3_siso_tpu_amd import _lib as lib

    h = lib.load()
    for entry in (h.m3s_embed_fwd, h.m3s_embed_bwd):
        assert entry(None, None) == lib.ERR_INVALID and b"NULL" in h.m3s_last_error()
        a = lib.EmbedArgs()
        a.struct_size = 3
        assert entry(ctypes.byref(a), None) == lib.ERR_INVALID and b"ABI mismatch" in h.m3s_last_error()

    def args(**kw):
        a = lib.EmbedArgs()
        a.struct_size, a.dtype, a.id_bytes = ctypes.sizeof(lib.EmbedArgs), lib.DTYPE_F32, 8
        a.vocab, a.width, a.tokens, a.padding_idx, a.table_stride = 10, 4, 6, -1, 4
        a.ids = a.table = a.y = a.dy = a.dtable = a.workspace = 4096   # never read: every call is refused
        a.workspace_bytes = h.m3s_embed_bwd_workspace_bytes(6, 10, 4)
        for k, v in kw.items():
            setattr(a, k, v)
        return a

    both = [dict(dtype=7), dict(id_bytes=2), dict(vocab=0), dict(width=0), dict(tokens=-1),
            dict(tokens=1 << 31), dict(width=1 << 22), dict(ids=None), dict(ids=4097)]
    for bad in both + [dict(table=None), dict(y=None), dict(table=4098), dict(table_stride=-1)]:
        assert h.m3s_embed_fwd(ctypes.byref(args(**bad)), None) == lib.ERR_INVALID, bad
    for bad in both + [dict(dy=None), dict(dtable=None), dict(dtable=4098), dict(workspace=None),
                       dict(workspace=4104), dict(workspace_bytes=args().workspace_bytes - 1)]:
        assert h.m3s_embed_bwd(ctypes.byref(args(**bad)), None) == lib.ERR_INVALID, bad
    assert h.m3s_embed_fwd(ctypes.byref(args(tokens=0)), None) == lib.OK   # nothing to launch
    for sizes in ((-1, 10, 4), (6, 0, 4), (6, 10, 0), (1 << 31, 10, 4)):
        assert h.m3s_embed_bwd_workspace_bytes(*sizes) == -1


def test_embed_struct_matches_the_header(m3, tmp_path):
    import os
    import subprocess

    from mamba3_siso_tpu_amd import _lib as lib

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src, exe = tmp_path / "t.c", tmp_path / "t"
    pairs = [("m3s_embed_args", lib.EmbedArgs)]
    lines = []
    for name, cls in pairs:
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        lines += [f'printf("%zu\\n", offsetof({name}, {f[0]}));' for f in cls._fields_]
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "m3s.h"\nint main(void) {\n'
                   + "\n".join(lines) + "\nreturn 0;\n}\n")
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    want = []
    for _, cls in pairs:
        want.append(ctypes.sizeof(cls))
        want += [getattr(cls, f[0]).offset for f in cls._fields_]
    assert got == want
