"""What kernels rely on and no run on a whole GPU shows when it is missing, read from the sources."""

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "tessiq_b200" / "csrc"
SOURCES = sorted(CSRC.glob("*.cu"))
DECLARED = re.compile(r"extern __shared__\s+(__align__\(\d+\)\s+)?((?:unsigned\s+)?\w+)\s+(\w+)\[\];")


@pytest.mark.parametrize("source", SOURCES, ids=lambda path: path.name)
def test_dynamic_shared_memory_is_aligned_by_what_declares_it(source):
    """Where it begins behind a kernel's static arrays is their sizes' accident: it says its alignment, is of vectors, or is rounded up where it is used."""
    text = source.read_text()
    for aligned, element, name in DECLARED.findall(text):
        assert aligned or element == "uint4" or re.search(rf"smem_address\({name}\) \+ \d+u\) & ~\d+u", text), f"{source.name}: {element} {name}[]"


@pytest.mark.parametrize("source", SOURCES, ids=lambda path: path.name)
def test_clusters_that_not_every_gpu_has_room_for_are_asked_about(source):
    """Clusters over eight are not portable: a part of a GPU, or one whose processing clusters have fewer multiprocessors, runs none of them."""
    text = source.read_text()
    if "cudaFuncAttributeNonPortableClusterSizeAllowed" in text:
        assert "cudaOccupancyMaxActiveClusters" in text
