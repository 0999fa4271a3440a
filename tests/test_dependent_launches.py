"""Kernels that start before the launch ahead of them has ended (programmatic dependent launch): what their sources may not say.

Such a kernel reads what the earlier launch writes while both run.  A read-only load (__ldg), a pointer that promises no other
access (__restrict__) or a load intrinsic outside the order of the wait may be moved ahead of the wait; the fault would
show now and then and not in a test of values, so this one reads the sources."""
import os
import re

import pytest

from conftest import ROOT

CSRC = os.path.join(ROOT, "stlq_b200", "csrc")


def code(name):
    """The file without its comments."""
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*|/\*.*?\*/", "", f.read(), flags=re.S)


def dependent():
    """The files that launch kernels so."""
    return sorted(n for n in os.listdir(CSRC) if n.endswith(".cu") and re.search(r"\bLaunchAfter\(|ProgrammaticStreamSerialization", code(n)))


def test_the_files_are_found():
    assert {"matmul_i8.cu", "routed.cu"} <= set(dependent())


@pytest.mark.parametrize("word", ["__ldg", "__ldcs", "__ldca", "__ldcg", "__ldlu", "__restrict__", "__restrict", "ld.global.nc"])
@pytest.mark.parametrize("name", dependent())
def test_no_claim_that_memory_is_read_only(name, word):
    assert not re.search(re.escape(word) + r"\b", code(name))


@pytest.mark.parametrize("name", dependent())
def test_every_kernel_waits_once(name):
    """Each kernel of these files calls WaitForEarlier, so that 'everything earlier has finished' holds along a chain of launches."""
    bodies = re.split(r"\b__global__\b", code(name))[1:]
    assert bodies and all(b.split("__global__")[0].count("WaitForEarlier();") == 1 for b in bodies)


def test_no_wait_of_the_products_gives_up_for_an_earlier_call():
    """The handle's error word outlives a call.  A wait that gives up because the word is raised would spoil every later product until
    someone asks for the error, so the products wait without looking at it (the last argument of MbarWait)."""
    calls = re.findall(r"\bMbarWait\(([^;]*)\);", code("matmul_i8.cu"))
    assert calls and all(c.rstrip().endswith(", false") for c in calls)


def test_errors_are_taken_in_one_step():
    """A word that is read, waited for and cleared loses what a kernel on another stream raises in between."""
    body = re.search(r"int stlq_b200_kernels_sync\(.*?\n}\n", code("provider.cu"), flags=re.S).group(0)
    assert "cudaMemset" not in body and "atomicExch(word, 0u)" in code("provider.cu")
