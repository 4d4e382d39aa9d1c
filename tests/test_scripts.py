"""The scripts of scripts/: what may be in them, and that the documents name only those that are there.

A build whose kernels fault or hang on the GPU is not run there again to narrow the failure down: the cause is looked for on the CPU (tests/wavemu executes the kernel source,
tests/isaemu the kernel binary).  So no GPU script may be one that does it."""
import glob
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FOLDERS = [os.path.join(ROOT, "scripts", d) for d in ("", "archive", "calib")]
GPU_SCRIPTS = sorted(p for d in FOLDERS for p in glob.glob(os.path.join(d, "gpu_*")))
DOCUMENTS = [os.path.join(ROOT, f) for f in ("README.md", "DESIGN.md", "INTEGRATION.md")] + sorted(glob.glob(os.path.join(ROOT, "profiles", "*.md")) + glob.glob(os.path.join(ROOT, "profiles", "*.txt")))
FAULT_WORDS = re.compile(r"\b(faults?|faulted|faulting|aborts?|aborted|hangs?|hung|crash\w*)\b", re.I)
FAILED_BUILDS = re.compile(r"libhpt_(prodfail|debugra|noslp|nosv|wait0|cw3|runB)\b|Memory access fault")


def explanations(text):
    """the comment lines and the docstring of a script"""
    doc = re.findall(r'"""(.*?)"""', text, re.S)
    return "\n".join([l for l in text.splitlines() if l.lstrip().startswith("#")] + doc)


@pytest.mark.parametrize("path", GPU_SCRIPTS, ids=os.path.basename)
def test_no_gpu_script_is_there_to_make_a_failure_happen_again(path):
    text = open(path).read()
    assert not FAULT_WORDS.search(explanations(text)), explanations(text)
    assert not FAILED_BUILDS.search(text)


def test_no_switch_of_the_product_builds_a_kernel_that_is_known_to_fault():
    for path in glob.glob(os.path.join(ROOT, "pbrt-v2_amd", "csrc", "*")) + [os.path.join(ROOT, "pbrt-v2_amd", "Makefile")]:
        assert "HPT_REGEN_ALL" not in open(path).read(), path          # the batched refill in the free-running kernels


def test_no_source_writes_packed_fp32_arithmetic_by_hand():
    """v_pk_add_f32 and its kind have given wrong results on the GPU now and then, without an error: no inline assembly issues them, in the product or beside it"""
    sources = [p for d in ("pbrt-v2_amd/csrc", "scripts/calib", "tests/isaemu/battery") for p in glob.glob(os.path.join(ROOT, d, "*")) if os.path.isfile(p)]
    assert len(sources) > 30
    for path in sources:
        for line in open(path, errors="replace"):
            if "asm" in line or "scripts" in path:
                assert not re.search(r"v_pk_(add|mul|fma)_f32", line), (path, line)


def test_documents_name_only_scripts_that_are_in_the_tree():
    missing = set()
    for doc in DOCUMENTS:
        for name in re.findall(r"scripts/[\w./]+?\.(?:sh|py|hip|cpp)\b|\bgpu_\w+\.(?:sh|py)\b", open(doc, errors="replace").read()):
            if not any(os.path.exists(os.path.join(d, os.path.basename(name))) for d in FOLDERS):
                missing.add((os.path.relpath(doc, ROOT), name))
    assert not missing, sorted(missing)


@pytest.mark.parametrize("path", GPU_SCRIPTS, ids=os.path.basename)
def test_no_gpu_script_repeats_a_test_to_see_whether_it_fails_again(path):
    """passes of another build say nothing about the one that failed, and a loop that drops the exit status does not stop at the first failure"""
    text = open(path).read()
    for loop in re.findall(r"^for (?:i|rep) in [\d ]+; do(.*?)^done", text, re.S | re.M):
        assert "pytest" not in loop, loop
