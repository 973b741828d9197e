"""Static checks of the product kernels' machine code (no GPU needed; hipcc cross-compiles).

The first waits of a block leave the stores of the block before in flight, by number: a wave's epilogue has to issue at least
that many behind the DMA instructions of the next block's first tiles (`young` in vql_product_kernel).  The 16-bit kernels
store past the caches where rows are whole 64-byte runs, which a compiler may quietly turn into ordinary stores.  And the
accumulators leave few registers: a spill in the loop, or a wait for the DMA in flight before a fragment is read, costs more
than any other mistake there could.
"""
import os
import re
import subprocess

import pytest

from conftest import ROOT
from vq_vae_amd.build import FLAGS

TYPES = {"bf16": 2, "f32": 4}


@pytest.fixture(scope="module", params=list(TYPES))
def kernels(request, tmp_path_factory):
    """(template arguments, element size, instructions) of every product kernel of one element type."""
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    if not os.path.exists(hipcc):
        pytest.skip("hipcc not available")
    out = tmp_path_factory.mktemp("isa") / "linear.s"
    src = os.path.join(ROOT, "vq_vae_amd", "csrc", f"vq_linear_{request.param}.hip")
    subprocess.check_call([hipcc, *FLAGS, "-S", "--cuda-device-only", "-o", str(out), src], stderr=subprocess.DEVNULL)
    text = out.read_text()
    found = []
    for m in re.finditer(r"^(_ZN\S*vql_product_kernelI\S*):", text, re.M):
        numbers = [int(v) for v in re.findall(r"L[bi](\d+)E", m.group(1))]
        body = text[m.end(): text.index(".end_amdhsa_kernel", m.end())]
        ops = [line.split(";")[0].strip() for line in body.split("\n")]
        found.append((numbers, TYPES[request.param], [op for op in ops if op and (op[0] != "." or op.startswith(".LBB"))]))
    assert len(found) == 25        # 3 epilogues of the forward pass and 2 gradients, 5 tiles each
    return found


def shape(numbers):
    a_major, b_major, kind, bi, bj, wi, wj, stages, dma = numbers
    return kind, (bi // wi // 32) * (bj // wj // 32), bool(dma)


def test_neither_spills_nor_flat_accesses(kernels):
    for numbers, _, ops in kernels:
        assert not [op for op in ops if op.startswith(("scratch_", "flat_"))], numbers


def test_stores_of_an_epilogue(kernels):
    for numbers, size, ops in kernels:
        kind, tiles, _ = shape(numbers)
        stores = tiles * size * (1 if kind == 0 else 2)          # 16-byte stores of the output and of what is kept for the activation
        past = [op for op in ops if op.startswith("global_store_dwordx4") and op.endswith(" nt")]
        others = [op for op in ops if op.startswith("global_store_dwordx4") and not op.endswith(" nt")]
        assert len(past) == (stores if size == 2 else 0), numbers
        # ordinary rows, a split sum's registers, and the blocks at the edge (which are not counted on)
        assert len(others) >= stores + 4 * tiles, numbers


def test_fragments_are_read_without_waiting_for_the_dma(kernels):
    for numbers, _, ops in kernels:
        _, _, dma = shape(numbers)
        if not dma:
            continue
        # the loop: from the first product's label to the last product
        products = [i for i, op in enumerate(ops) if op.startswith("v_mfma")]
        last_label = max(i for i in range(products[0]) if ops[i].startswith(".LBB"))
        loop = ops[last_label: products[-1]]
        assert any(op.startswith("buffer_load") and op.endswith(" lds") for op in loop), numbers
        for i, op in enumerate(loop):
            if op.startswith("s_waitcnt") and "vmcnt" in op:
                # only in the barrier's own waits: no product and no fragment read before the barrier
                rest = next((o for o in loop[i + 1:] if o.startswith(("v_mfma", "ds_read", "s_barrier", "global_load", "ds_write"))), "s_barrier")
                assert rest == "s_barrier" or rest.startswith(("ds_write", "global_load")), (numbers, op, rest)
