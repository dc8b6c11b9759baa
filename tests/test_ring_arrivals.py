"""Arrivals on the barriers that free a ring's buffers: the tensor core makes them (tcgen05.commit) whenever it gets there, and one
that nobody waits for may come when its CTA has ended.  Shown without a GPU: that a late arrival would fault one."""
import os
import re
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "lfm25-inference_b200", "csrc")

PROGRAM = r"""
#include <cstdio>
#include <vector>
#include "ring.h"

// The producer of a ring waits for a buffer's arrival before it fills it again; the consumer arrives where `filled_again`
// says so.  Every arrival is waited for, and every wait has its arrival.
int main() {
    for (unsigned buffers = 1; buffers < 9; ++buffers) {
        for (unsigned items = 0; items < 40; ++items) {
            std::vector<unsigned> arrivals(buffers, 0), waits(buffers, 0);
            for (unsigned index = 0; index < items; ++index) {
                if (index >= buffers) ++waits[index % buffers];
                if (lfm25::filled_again(index, items, buffers)) ++arrivals[index % buffers];
            }
            if (arrivals != waits) {
                std::printf("%u items in %u buffers\n", items, buffers);
                return 1;
            }
        }
    }
    // sets that take items by turns wait once each, for their last item
    for (unsigned sets = 1; sets < 4; ++sets) {
        for (unsigned items = 0; items < 40; ++items) {
            std::vector<unsigned> reports(sets, 0), waits(sets, 0);
            for (unsigned index = 0; index < items; ++index) {
                if (lfm25::last_of_set(index, items, sets)) ++reports[index % sets];
            }
            for (unsigned set = 0; set < sets; ++set) waits[set] = items > set ? 1 : 0;
            if (reports != waits) {
                std::printf("%u items, %u sets\n", items, sets);
                return 1;
            }
        }
    }
    std::puts("ok");
    return lfm25::filled_again(0xfffffff0u, 0xffffffffu, 15) ? 1 : 0;   // no sum that wraps
}
"""


def test_a_buffer_is_reported_free_as_often_as_it_is_filled_again(tmp_path):
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    source = tmp_path / "ring.cpp"
    source.write_text(PROGRAM)
    binary = tmp_path / "ring"
    compiled = subprocess.run(["g++", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-I", CSRC, str(source), "-o", str(binary)],
                              capture_output=True, text=True)
    assert compiled.returncode == 0, compiled.stderr
    ran = subprocess.run([str(binary)], capture_output=True, text=True, timeout=60)
    assert ran.returncode == 0 and ran.stdout.strip() == "ok", ran.stdout


@pytest.mark.parametrize("name", ["stack_attention_umma.cu", "hybrid_attention_umma.cu", "stack_latent_decode.cu", "e4m3_attention_umma.cu", "gemm_rows_umma.cu", "fp8_gemm_umma.cu"])
def test_kernels_ask_for_arrivals_that_are_waited_for(name):
    with open(os.path.join(CSRC, name)) as handle:
        commits = [line.strip() for line in handle if re.search(r"umma_commit\(bar_empty", line)]
    assert commits and all(line.startswith("if (filled_again(") for line in commits), commits


def test_every_product_of_the_prompt_attention_is_waited_for():
    """One set of softmax warps waits for every stage's product in turn; of two sets each waits for its last stage's, and no other
    is reported."""
    with open(os.path.join(CSRC, "e4m3_attention_umma.cu")) as handle:
        source = handle.read()
    commits = re.findall(r"^ *(.*umma_commit\(my_product.*)$", source, re.M)
    assert commits == ["if (kSets == 1 || last_of_set(stage, my_stages, kSets)) umma_commit(my_product + 8 * parity);"]
    loop = source[source.index("for (uint32_t stage = set; stage < my_stages; stage += kSets)"):]
    assert re.search(r"if \(kSets == 1 && stage >= 2\) \{\s*ok = ok && mbar_wait_bounded\(bar_product", loop)


def test_every_product_of_the_latent_decode_attention_is_waited_for():
    """Stage `index` waits for the product of index - 2, and the end for the last two."""
    with open(os.path.join(CSRC, "stack_latent_decode.cu")) as handle:
        source = handle.read()
    assert len(re.findall(r"umma_commit\(bar_product", source)) == 1
    assert re.search(r"if \(index >= 2\) \{\s*ok = mbar_wait_bounded\(bar_product \+ 8 \* buffer", source)
    end = source[source.index("const uint32_t last = count - 1;"):]
    assert re.search(r"bar_product \+ 8 \* \(\(last - 1\) & 1\)", end) and re.search(r"bar_product \+ 8 \* \(last & 1\)", end)


def test_every_block_of_the_f32_product_is_waited_for():
    """Waited for are: by the producer blocks whose slot is filled again, by the adding warps the later block of each pair, by the issuing
    lane the earlier ones of the pairs that are left."""
    with open(os.path.join(CSRC, "linear_f32.cu")) as handle:
        source = handle.read()
    issuing = source[source.index("umma_commit(bar_read"):source.index("} else if (warp < kFirstAdder)")]
    assert "unfilled = blocks > S::kStages ? blocks - S::kStages : 0;" in issuing
    assert re.search(r"first = \(unfilled \+ 1\) & ~1u; block == blocks && first \+ 1 < blocks; first \+= 2\) \{\s*\(void\)mbar_wait_bounded\(bar_read",
                     issuing)
    for stages in (3, 4, 5):
        for blocks in range(1, 40):
            unfilled = max(blocks - stages, 0)
            waited = set(range(unfilled)) | {min(pair + 1, blocks - 1) for pair in range(0, blocks, 2)}
            waited |= set(range((unfilled + 1) & ~1, blocks - 1, 2))
            assert waited == set(range(blocks)), (blocks, stages)
