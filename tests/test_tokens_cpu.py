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
    for bad in (table[0], table[0, 0]):
        with pytest.raises(ValueError, match="must be \\(V, D\\)"):
            m3.embed_tokens(bad, tokens, padding_idx=0)
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
        a.vocab, a.width, a.tokens, a.padding_idx, a.table_stride = 10, 4, 2000, -1, 4
        a.ids = a.table = a.y = a.dy = a.dtable = a.workspace = 4096   # never read: every call is refused
        a.workspace_bytes = h.m3s_embed_bwd_workspace_bytes(2000, 10, 4)
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
    assert h.m3s_embed_bwd_workspace_bytes(1024, 10, 4) == 0   # few tokens are not sorted
    assert h.m3s_embed_bwd_workspace_bytes(1025, 10, 4) > 0
    assert h.m3s_embed_bwd_workspace_bytes(1024, 1 << 20, 64) == 0
    assert h.m3s_embed_bwd_workspace_bytes(1024, 1 << 20, 65) > 0


def test_structs_match_the_header(m3, tmp_path):
    import os
    import subprocess

    from mamba3_siso_tpu_amd import _lib as lib

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src, exe = tmp_path / "t.c", tmp_path / "t"
    pairs = [("m3s_embed_args", lib.EmbedArgs), ("m3s_logprob_args", lib.LogprobArgs),
             ("m3s_distill_args", lib.DistillArgs)]
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


def test_logprobs_and_distillation_refuse_bad_arguments(m3):
    x, t = torch.zeros(3, 10), torch.zeros(3, dtype=torch.int64)
    ids, u = torch.zeros(3, 4, dtype=torch.int64), torch.zeros(3, 4)
    T, D = m3.token_logprobs, m3.distill_loss
    for call in (lambda: T(x, t), lambda: D(x, ids, u)):
        with pytest.raises(ValueError, match="ROCm device only"):
            call()
    for top in (-1, 11, 65):
        with pytest.raises(ValueError, match="top must be"):
            T(torch.zeros(3, 100) if top == 65 else x, t, top=top)
    for temp in (0.0, -1.0, float("nan"), float("inf")):
        for call in (lambda: T(x, t, temperature=temp), lambda: D(x, ids, u, temperature=temp)):
            with pytest.raises(ValueError, match="temperature"):
                call()
    bad = [lambda: T(x.double(), t), lambda: T(x, t.float()), lambda: T(x, t[:2]), lambda: T(x[:, :0], t),
           lambda: T(torch.tensor(1.0), t), lambda: T(x, t[:, None]),
           lambda: D(x.half(), ids, u), lambda: D(x, ids[:2], u), lambda: D(x, ids, u[:, :3]),
           lambda: D(x, ids.short(), u), lambda: D(x, ids, u.double()), lambda: D(x, ids[:, :0], u[:, :0]),
           lambda: D(x, ids.repeat(1, 65), u.repeat(1, 65)), lambda: D(x, ids, u, targets=t[:1]),
           lambda: D(x, ids, u, targets=t.bool()), lambda: D(x, ids[0], u[0])]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    with pytest.raises(ValueError, match="must not require a gradient"):
        D(x, ids, u.requires_grad_(True))
    K, stats3, stats5 = m3.kernels, torch.zeros(3, 3), torch.zeros(3, 5)
    with pytest.raises(ValueError, match="needs the targets"):
        K.logprob_backward(x, None, stats3, dlogp=torch.zeros(3))
    with pytest.raises(ValueError, match="needs top_ids"):
        K.logprob_backward(x, t, stats3, dtop_logp=torch.zeros(3, 2))
    with pytest.raises(ValueError, match="stats"):
        K.logprob_backward(x, t, stats5, dlogp=torch.zeros(3))


def test_vocab_abi_refuses_bad_structs(m3):
    from mamba3_siso_tpu_amd import _lib as lib

    h = lib.load()
    entries = ((h.m3s_logprob_fwd, lib.LogprobArgs), (h.m3s_logprob_bwd, lib.LogprobArgs),
               (h.m3s_distill_fwd, lib.DistillArgs), (h.m3s_distill_bwd, lib.DistillArgs))

    def args(cls, **kw):
        a = cls()
        a.struct_size, a.dtype = ctypes.sizeof(cls), lib.DTYPE_F32
        a.batch, a.seqlen, a.vocab, a.temperature, a.ignore_index = 2, 3, 10, 1.0, -100
        a.logits = lib.Blx(4096, 30, 10)   # addresses are never read: every call is refused
        for name in ("targets", "stats", "dlogits"):
            setattr(a, name, 4096)
        if cls is lib.LogprobArgs:
            a.top = 2
            for name in ("logp", "entropy", "top_logp", "top_ids", "dlogp", "dtop_logp"):
                setattr(a, name, 4096)
        else:
            a.teacher_k, a.id_bytes, a.teacher_dtype = 4, 8, lib.DTYPE_BF16
            for name in ("teacher_ids", "teacher_logits", "kd", "nll", "dkd", "dnll"):
                setattr(a, name, 4096)
        for k, v in kw.items():
            setattr(a, k, v)
        return a

    common = [dict(dtype=5), dict(batch=-1), dict(seqlen=-1), dict(vocab=0), dict(vocab=1 << 30),
              dict(batch=1 << 16, seqlen=1 << 16), dict(temperature=0.0), dict(temperature=-2.0),
              dict(temperature=float("nan")), dict(temperature=float("inf")), dict(temperature=1e-39),
              dict(logits=lib.Blx(None, 30, 10)), dict(logits=lib.Blx(4098, 30, 10)),
              dict(logits=lib.Blx(4096, -30, 10)), dict(logits=lib.Blx(4096, 30, -10))]
    own = [[dict(top=-1), dict(top=65, vocab=100), dict(top=11), dict(logp=None), dict(entropy=None),
            dict(top_logp=None), dict(top_ids=None)],
           [dict(stats=None), dict(top=65, vocab=100), dict(dlogits=None), dict(dlogits=4098), dict(targets=None),
            dict(top_ids=None)],
           [dict(teacher_k=0), dict(teacher_k=257), dict(id_bytes=2), dict(teacher_dtype=9), dict(kd=None),
            dict(nll=None), dict(targets=None), dict(teacher_ids=None), dict(teacher_logits=None)],
           [dict(stats=None), dict(teacher_k=0), dict(dlogits=None), dict(dlogits=4098), dict(targets=None),
            dict(teacher_ids=None)]]
    for (entry, cls), extra in zip(entries, own):
        assert entry(None, None) == lib.ERR_INVALID and b"NULL" in h.m3s_last_error()
        assert entry(ctypes.byref(args(cls, struct_size=3)), None) == lib.ERR_INVALID
        assert b"ABI mismatch" in h.m3s_last_error()
        for bad in common + extra:
            assert entry(ctypes.byref(args(cls, **bad)), None) == lib.ERR_INVALID, (cls, bad)
        assert entry(ctypes.byref(args(cls, batch=0)), None) == lib.OK   # nothing to launch


def test_sizes_past_32_bits_are_refused(m3):
    """The args structs hold rows, vocabularies and widths in 32 bits: what is larger must not reach
    them cut short (2^32 + 5 ids would become 5)."""
    one, t = torch.zeros(1, 1), torch.zeros(3, dtype=torch.int64)
    K = m3.kernels
    for shape in ((2 ** 32 + 5, 1), (2 ** 31 - 1, 1), (1, 2 ** 32 + 4), (1, 2 ** 22)):
        with pytest.raises(ValueError, match="too large"):
            m3.embed_tokens(one.expand(shape), t)
        with pytest.raises(ValueError, match="too large"):
            K.embedding_backward(t, one[0].expand(3, shape[1]), shape[0])
    with pytest.raises(ValueError, match="too large"):
        m3.embed_tokens(torch.zeros(5, 4), t[:1].expand(2 ** 31))
    assert K.embedding_fits(2 ** 31 - 2, 2 ** 22 - 1, 2 ** 31 - 65)
    for shape in ((2 ** 32 + 3, 1), (2 ** 32, 3, 1), (3, 2 ** 32, 1), (2 ** 16, 2 ** 16, 4), (2 ** 31, 2), (1, 2 ** 32 + 8),
                  (2, 2 ** 30)):
        x = one.view(-1).expand(shape)
        with pytest.raises(ValueError, match="fewer than 2\\^31"):
            m3.token_logprobs(x, t)
        with pytest.raises(ValueError, match="fewer than 2\\^31"):
            m3.distill_loss(x, t[:, None], torch.zeros(3, 1))


def test_node_module_is_checked_at_load(m3, tmp_path, monkeypatch):
    """A missing module of nodes and one of another torch raise; its calls refuse other arguments."""
    from mamba3_siso_tpu_amd import _lib as lib

    mod = lib.nodes()
    assert mod is lib.nodes() and mod.torch_version == torch.__version__.split("+")[0]
    for call in (lambda: mod.embed(torch.zeros(2, 2)), lambda: mod.bind(1)):
        with pytest.raises(TypeError):
            call()
    # what is not the node's: tensors on the CPU, and no tensors at all
    assert mod.embed(torch.zeros(2, 2), torch.zeros(1, dtype=torch.int64), 1.0, -1, False) is None
    assert mod.embed(None, [1], 1.0, -1, False) is None
    monkeypatch.setattr(lib, "_nodes", None)
    with pytest.raises(RuntimeError, match="missing"):
        lib.nodes(str(tmp_path / "m3s_nodes.so"))
    broken = tmp_path / "m3s_nodes.so"
    broken.write_bytes(b"not a library")
    with pytest.raises(RuntimeError, match="rebuild"):
        lib.nodes(str(broken))
    monkeypatch.setattr(torch, "__version__", "1.0.0+other")
    with pytest.raises(RuntimeError, match="rebuild"):
        lib.nodes()


def test_distill_step_refuses_k_when_it_is_built(m3):
    """The teacher's pass leaves at most 64 tokens: another k is refused before the teacher has run."""
    cfg = m3.model.LMConfig(vocab_size=100, n_layers=1, siso=m3.SISOConfig(d_model=64, d_state=16, headdim=16))
    small = m3.model.LMConfig(vocab_size=40, n_layers=1, siso=cfg.siso)
    for k in (0, -1, 65, 100, 1000):
        with pytest.raises(ValueError, match="k must be in"):
            m3.train.make_distill_step(cfg, None, None, cfg, k=k)
    for k, c in ((1, cfg), (64, cfg), (100, small)):
        assert callable(m3.train.make_distill_step(c, None, None, c, k=k))
