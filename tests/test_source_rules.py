"""Rules over the source text that no run shows: each guards against a way of building or driving
the GPU that has failed without an error of its own (a hang, a fault, a wrong sum now and then)."""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _sources(*tops, ext=(".hip", ".h", ".cpp", ".py", ".sh", ".c", "Makefile")):
    """(path relative to the root, text) of every source file under the given folders or files"""
    out = []
    for top in tops:
        p = os.path.join(ROOT, top)
        names = [p] if os.path.isfile(p) else [os.path.join(d, f) for d, _, fs in os.walk(p) for f in fs]
        for n in names:
            if n.endswith(ext) and os.path.abspath(n) != os.path.abspath(__file__):
                with open(n, encoding="utf-8") as f:
                    out.append((os.path.relpath(n, ROOT), f.read()))
    assert out
    return out


def test_every_stream_has_the_default_priority():
    """Work on streams of different priorities beside each other can hang the device."""
    bad = re.compile(r"hipStreamCreateWithPriority|cudaStreamCreateWithPriority|StreamPriorityRange|"
                     r"is_high_priority_stream|Stream\([^)]*priority")
    hits = ["%s: %s" % (n, m.group(0)) for n, t in _sources("veneur_amd", "include", "tools", "tests", "bench.py",
                                                           "__graft_entry__.py") for m in bad.finditer(t)]
    assert not hits, hits


def test_no_build_selects_the_division_that_faulted():
    """A build whose replays divide with ddiv_nr gave wrong digests and GPU faults, cause unproven:
    no macro selects it, and only the diagnostic entry instantiates it."""
    src = _sources("veneur_amd", "include", ext=(".hip", ".h", ".cpp", ".py", "Makefile"))
    assert not [n for n, t in src if re.search(r"VN_INDEX_NR|VN_NR_", t)]
    uses = [(n, m.group(0)) for n, t in src for m in re.finditer(r"(index_estimate|asin_go_sel)<(?!false)[^>]*>", t)]
    assert uses == [("veneur_amd/csrc/capi.hip", "index_estimate<true>"), ("veneur_amd/csrc/gomath.h", "asin_go_sel<NR>")]
    decl = [t for n, t in src if n.endswith("gomath.h")][0]
    assert re.findall(r"template <bool NR[^>]*>", decl) == ["template <bool NR = false>"] * 2


def test_tools_repeat_no_failing_case():
    """The tools measure; they run no test's case in a loop, select no build with recorded faults
    and read no log for a fault to go on after it.  What they run is in the tree."""
    src = [(n, t) for n, t in _sources("tools", "bench.py") if not n.endswith((".hip", ".c"))]
    bad = re.compile(r"from tests\.test_|import tests\.test_|libveneur_amd_nr|Memory access fault|illegal memory access|"
                     r"\bFAILED\b")
    assert not ["%s: %s" % (n, m.group(0)) for n, t in src for m in bad.finditer(t)]
    named = re.compile(r"(?<![\w/.])((?:tools|tests)/[\w/]+\.(?:py|sh|hip|c))\b")
    assert not ["%s: %s" % (n, p) for n, t in src for p in named.findall(t) if not os.path.exists(os.path.join(ROOT, p))]


def test_device_code_is_built_without_packed_fp32():
    """Some forms of the packed FP32 instructions, which the compiler makes from ordinary float
    code, have given wrong results now and then: every HIP compile line turns them off."""
    flag = "-Xclang -target-feature -Xclang -packed-fp32-ops"
    (_, mk), = _sources("veneur_amd/Makefile")
    assert "NO_PACKED_FP32 := " + flag in mk
    lines = [ln for ln in mk.splitlines() if "$(HIPCC)" in ln and " -c " in ln]
    assert lines and all("$(CXXFLAGS)" in ln for ln in lines)
    assert re.search(r"^CXXFLAGS \?= (.*\\\n)*.*\$\(NO_PACKED_FP32\)", mk, re.M)
    hip = _sources("veneur_amd", "tools", "include", ext=(".hip", ".h"))
    assert not [n for n, t in hip for ln in t.splitlines() if "Build: hipcc" in ln and flag not in ln]
    assert not [n for n, t in hip if re.search(r"v_pk_(add|mul|fma)_f32", t)]
