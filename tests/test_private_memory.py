"""A kernel with private memory (spilled registers) needs device memory that the
runtime looks for at its launch, a few hundred MB at 440 bytes a lane; where there
is none it ends the process, which no call can report.  The kernels of a training step have
none: their metadata in the built library says so."""
import os
import re
import subprocess

import pytest

from burn_dragon_amd import build

LLVM = "/opt/rocm/llvm/bin"


def _run(*args):
    r = subprocess.run(args, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-1000:]
    return r.stdout


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """{kernel: (bytes of private memory a lane, spilled vector registers)} of the library."""
    tools = [os.path.join(LLVM, t) for t in ("llvm-objcopy", "clang-offload-bundler", "llvm-readelf")]
    if not os.path.exists(build.LIB) or not all(os.path.exists(t) for t in tools):
        pytest.skip("no built library, or no tools to read it")
    objcopy, bundler, readelf = tools
    d = str(tmp_path_factory.mktemp("kernels"))
    fat, found = os.path.join(d, "fat"), {}
    _run(objcopy, f"--dump-section=.hip_fatbin={fat}", build.LIB, os.path.join(d, "copy"))
    data = open(fat, "rb").read()
    magic = b"__CLANG_OFFLOAD_BUNDLE__"
    starts = [m.start() for m in re.finditer(magic, data)] + [len(data)]
    for i, (a, b) in enumerate(zip(starts, starts[1:])):  # one of each source file
        part, elf = os.path.join(d, f"part{i}"), os.path.join(d, f"elf{i}")
        open(part, "wb").write(data[a:b])
        _run(bundler, "--unbundle", "--type=o", f"--input={part}", f"--output={elf}",
             f"--targets=hipv4-amdgcn-amd-amdhsa--{build.ARCH}")
        for k in _run(readelf, "--notes", elf).split("- .agpr_count:")[1:]:
            get = lambda key: re.search(rf"\.{key}:\s+(\S+)", k).group(1)  # noqa: E731
            found[get("name")] = int(get("private_segment_fixed_size")), int(get("vgpr_spill_count"))
    assert found
    return found


@pytest.mark.parametrize("part,least", [("gated_kernel", 48), ("few_kernel", 48), ("fused_kernel", 8), ("product_kernel", 4),
                                        ("gated_grads_kernel", 3), ("join_kernel", 1), ("embed_", 20), ("sort_small_kernel", 1),
                                        ("digit_", 4), ("save_kernel", 2), ("restore_kernel", 2)])
def test_kernels_of_a_training_step_have_no_private_memory(kernels, part, least):
    mine = {k: v for k, v in kernels.items() if part in k}
    assert len(mine) >= least
    assert not {k: v for k, v in mine.items() if v != (0, 0)}
