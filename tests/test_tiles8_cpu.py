"""The index rules of the tiled products in 8 bits (``csrc/m3s_tiles8.h``), compiled for the host and held
to the sizes of what they point into: a value that the kernel reads and throws away shows in no result."""

import os
import subprocess
import sys

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mamba3-siso-tpu_amd", "csrc")


def run(tmp_path, body):
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text('#include <stdio.h>\n#include "m3s_tiles8.h"\nusing namespace m3s;\nint main() {\n' + body + "\n}\n")
    subprocess.run([os.environ.get("CXX", "g++"), "-O1", "-std=c++17", "-Wall", "-Werror", "-I", CSRC, str(src), "-o", str(exe)],
                   check=True, stdout=sys.stderr)
    return subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout


@pytest.mark.parametrize("tile_groups", [2, 4])
def test_scales_of_a_weight_are_read_within_it(tmp_path, tile_groups):
    """Every group of a tile of outputs, the last one's groups behind the weight too, every lane and every
    step that is asked for, three behind the last."""
    out = run(tmp_path, f"""
  long bad = 0, calls = 0;
  for (int np = 64; np <= 2048; np += 64)
    for (int kb = 1; kb <= 5; ++kb) {{
      const long bytes = (long)kb * np * 4;
      const int groups = np / 64;
      for (int g0 = 0; g0 < groups; g0 += {tile_groups})
        for (int q = 0; q < {tile_groups}; ++q)
          for (int entry = 0; entry < 32; ++entry)
            for (int s = 0; s < 2 * kb + 3; ++s) {{
              const int at = step_within(s, 2 * kb);
              const long byte = (long)weight_scale_at(g0 + q, groups, entry) + weight_scale_step(at, np);
              bad += at < 0 || at >= 2 * kb || byte < 0 || byte + 4 > bytes;
              // a group of the weight has its own scales: dword (step of 128, group, lane 16 g + r)
              const int g = 2 * (s & 1) + entry / 16;
              if (s < 2 * kb && g0 + q < groups) bad += byte != (((long)(s / 2) * groups + g0 + q) * 64 + 16 * g + entry % 16) * 4;
              ++calls;
            }}
    }}
  printf("%ld %ld\\n", bad, calls);""")
    bad, calls = map(int, out.split())
    assert bad == 0 and calls > 100000


def test_every_form_has_its_sizes(tmp_path):
    """The sizes that the GPU's tests take for a form take it, each form with whole pieces and an odd width."""
    import test_gpu_eight_forms as forms

    names = ["few16", "few32", "tiles64", "tiles64wide", "tiles128"]
    cases = [(f, r, -(-n // 64) * 64, n) for f, r, k, n in forms.each(forms.FORMS)]
    gated = [(f, r, -(-n // 128) * 256, n) for f, r, k, n in forms.each(forms.GATED_FORMS)]
    out = run(tmp_path, "".join(f'printf("%d ", (int)form8({r}, {np}));' for _, r, np, _ in cases + gated) + 'puts("");')
    assert [names[int(i)] for i in out.split()] == [c[0] for c in cases + gated]
    for some in (cases, gated):
        for f in names:
            widths = [n for name, _, _, n in some if name == f]
            assert any(n % 2 for n in widths) and any(n % 8 == 0 for n in widths), f


def test_one_rule_for_rows_rounded_in_the_launch():
    """The library's own answer, which both callers take: turns of workgroups on 256 CUs times a row's bytes."""
    from mamba3_siso_tpu_amd import _lib

    takes, bf16, f32 = _lib.load().m3s_matmul8_takes_floats, _lib.DTYPE_BF16, _lib.DTYPE_F32
    for rows, k, n, gated, dtype, want in (
            (1, 1024, 4480, 0, bf16, 1), (112, 1024, 4480, 0, bf16, 1), (160, 1024, 4480, 0, bf16, 1), (192, 1024, 4480, 0, bf16, 0),
            (80, 1024, 2816, 1, bf16, 1), (48, 2048, 4480, 0, bf16, 1), (96, 2048, 4480, 0, bf16, 0), (16, 2048, 32000, 0, bf16, 1),
            (17, 2048, 32000, 0, bf16, 0), (16, 4096, 2048, 0, bf16, 1), (17, 4096, 2048, 0, bf16, 0), (16, 4097, 2048, 0, bf16, 0),
            (48, 1024, 4480, 0, f32, 1), (64, 1024, 4480, 0, f32, 0), (8, 2048, 1024, 0, f32, 1), (9, 2048, 1024, 0, f32, 0),
            (256, 200, 1000, 0, bf16, 1), (257, 200, 1000, 0, bf16, 0), (0, 64, 64, 0, bf16, 1), (-1, 64, 64, 0, bf16, 0),
            (4, 0, 64, 0, bf16, 0), (4, 64, 0, 0, bf16, 0), (4, (1 << 20) + 1, 64, 0, bf16, 0), (4, 64, 64, 0, _lib.DTYPE_ROWS8, 0)):
        assert takes(rows, k, n, gated, dtype) == want, (rows, k, n, gated, dtype)
