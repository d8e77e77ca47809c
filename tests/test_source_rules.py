"""Rules that hold for the text of every source, script and build file of the tree (no GPU, no build needed)."""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DIRS = ("include", "liquid_cache_amd", "oracle", "scripts", "tests")
CODE = {".hip", ".cpp", ".hpp", ".c", ".h", ".s", ".S", ".py", ".sh"}


def code_files():
    walks = [(ROOT, [], [n for n in os.listdir(ROOT) if os.path.isfile(os.path.join(ROOT, n))])]
    for top in DIRS:
        walks += os.walk(os.path.join(ROOT, top))
    for d, _, names in walks:
        for n in names:
            if (os.path.splitext(n)[1] in CODE or n == "Makefile") and os.path.join(d, n) != os.path.abspath(__file__):
                yield os.path.join(d, n)


def matches(pattern):
    rx = re.compile(pattern)
    out = []
    for path in code_files():
        with open(path, encoding="utf-8", errors="replace") as f:
            for no, line in enumerate(f, 1):
                if rx.search(line):
                    out.append("%s:%d: %s" % (os.path.relpath(path, ROOT), no, line.strip()))
    return out


def test_the_walk_finds_the_kernels():
    found = {os.path.relpath(p, ROOT) for p in code_files()}
    assert {"liquid_cache_amd/csrc/lc_kernels.hip", "liquid_cache_amd/csrc/lc_runtime.cpp", "liquid_cache_amd/csrc/Makefile",
            "bench.py", "scripts/vgprs.sh"} <= found


# an instruction of the scalar unit with a store, an atomic or an operation on its data cache in its name; in inline assembly
# the escape of a newline or a tab may stand right before it
SCALAR_WRITE = r"(?:\b|\\[nt])s_(?:[a-z]+_)?(?:store|atomic|dcache)"


def test_device_code_writes_through_vector_stores_only():
    """Nothing writes through the scalar data cache: its lines are not coherent with the vector caches, and writing a wave's ballots
    that way took 1.75 times as long as v_writelane and a vector store (134 MB written: 223 against 127 us)."""
    assert matches(SCALAR_WRITE) == []


def test_every_stream_has_the_default_priority():
    """The index builder's stream and the streams of queries are busy at the same time; work on streams of different priorities
    may wait for good."""
    assert matches(r"StreamPriority|StreamCreateWithPriority|is_high_priority_stream|Stream\([^)]*\bpriority\s*=") == []


def test_tensors_are_exchanged_through_the_sharding_module():
    """torch.distributed's collectives on tensors are called in sharding.py alone, which gives gloo host memory only: its collectives
    on device tensors may hang when several ranks share one GPU."""
    calls = matches(r"\bdist\.(?:all_reduce|all_gather|all_to_all|reduce|broadcast|gather|scatter|send|recv|i(?:send|recv))\w*\(")
    assert [c for c in calls if not c.startswith("liquid_cache_amd/sharding.py:") and "_object" not in c] == []


def test_hip_code_is_compiled_without_packed_fp32():
    """The packed FP32 instructions are off wherever HIP code is compiled (hipcc makes them by itself from ordinary float code) and
    written nowhere by hand: some of their forms may give wrong results."""
    off = "-Xclang -target-feature -Xclang -packed-fp32-ops"
    with open(os.path.join(ROOT, "liquid_cache_amd", "csrc", "Makefile"), encoding="utf-8") as f:
        text = f.read()
    assert re.search(r"^DEVFLAGS := " + off + "$", text, re.M)
    compiles = [line for line in text.splitlines() if "$(HIPCC)" in line and " -c " in line]
    assert compiles and all("$(DEVFLAGS)" in line for line in compiles), compiles
    lines = [m for m in matches(r"hipcc --offload-arch") if "__graft_entry__" not in m and "_native.py" not in m]
    assert [m for m in lines if "packed-fp32-ops" not in m] == []
    assert matches(r"(?:\b|\\[nt])v_pk_(?:add|mul|fma)_f32") == []
