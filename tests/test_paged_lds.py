"""What the streaming attention's constants promise each other, at compile time (no GPU)."""
import subprocess

import pytest

from alveare_amd import build


def compiles(tmp_path, checks):
    """static_asserts over every variant of the streaming kernel: D, QT, E8 (8-bit pages)."""
    try:
        hipcc = build._hipcc()
    except RuntimeError:
        pytest.skip("no hipcc")
    src = tmp_path / "check.hip"
    src.write_text('#include "paged_attn.h"\nnamespace alv {\nnamespace {\ntemplate <int D, int QT, bool E8>\nstruct Check {\n'
                   + checks + "};\ntemplate <int D, int QT>\nstruct Both : Check<D, QT, false>, Check<D, QT, true> {};\n"
                   "[[maybe_unused]] Both<64, 1> a1;\n[[maybe_unused]] Both<64, 2> a2;\n[[maybe_unused]] Both<64, 4> a4;\n"
                   "[[maybe_unused]] Both<128, 1> b1;\n[[maybe_unused]] Both<128, 2> b2;\n[[maybe_unused]] Both<128, 4> b4;\n"
                   "[[maybe_unused]] Both<256, 1> c1;\n[[maybe_unused]] Both<256, 2> c2;\n[[maybe_unused]] Both<512, 1> d1;\n"
                   "}\n}\n")
    r = subprocess.run([hipcc, *build.HIPCC_FLAGS, "-Wno-everything", "-I", build.CSRC, "--offload-device-only", "-fsyntax-only",
                        str(src)], capture_output=True, text=True)
    assert r.returncode == 0, "\n".join(l for l in r.stderr.splitlines() if "error" in l or "note" in l)


def test_every_wave_has_a_flag(tmp_path):
    """Behind the rings, the waves' maxima and sums and q there is an int of LDS for each wave."""
    for two in ("false", "true"):
        compiles(tmp_path, f"""
    static constexpr int waves = rows_waves(D, {two});
    static constexpr int used = rows_mls(D, QT, E8, {two}) + 2 * waves * 16 * QT * 4 + (rows_q_lds(D, QT) ? 32 * QT * D : 0);
    static_assert(rows_lds(D, QT, E8, {two}) - used >= 4 * waves, "a flag for each wave");
    static_assert(used % 4 == 0, "aligned");
""")


def test_workgroups_that_share_a_cu_fit_its_lds(tmp_path):
    """The streaming kernel's grid counts on two workgroups a CU where rows_two says so, else on one."""
    compiles(tmp_path, """
    static_assert((rows_two(D, QT, E8) ? 2 : 1) * rows_lds(D, QT, E8, rows_two(D, QT, E8)) <= 160 * 1024, "LDS of a CU");
    static_assert(E8 || !rows_two(D, QT, E8), "bf16 rings are a CU's");
""")
