"""Bounded waits in front of code that takes a whole warp. A wait that gives up may do so in some lanes of a warp
alone. Where a vote, a shuffle or a tcgen05.ld / .st follows, the warp has to decide together, or it waits at the
vote for lanes that have left. Read off the sources: such a failure cannot be made on a GPU without a hang."""
import os
import re

from conftest import PKG


def source(name):
    text = open(os.path.join(PKG, "csrc", name)).read()
    return re.sub(r"//[^\n]*", "", text)


def test_softmax_warps_of_the_attention_kernel():
    text = source("flash_attn.cu")
    body = text[text.index("constexpr int KPT"):text.index("tmem_dealloc(tmem, C::TMEM_COLS)")]
    for call in ("mbar_wait(", "exchange("):
        uses = [m.start() for m in re.finditer(re.escape(call), body)]
        assert uses
        for at in uses:
            assert body[:at].endswith("together("), body[max(0, at - 80):at + 40]
    assert re.search(r"together = \[\]\(bool \w+\) \{ return __all_sync\(0xffffffffu", body)


def test_row_kernel_over_a_4_bit_cache():
    text = source("flash_attn_kvq.cu")
    body = text[text.index("kvq_rows_kernel("):text.index("kvq_join_kernel")]
    # the one wait outside a lone thread's branch is put to a vote at once
    assert re.search(r"const bool got = mbar_wait\(full\(stage\)[^;]*;\s*if \(__any_sync\(0xffffffffu, !got\)\) break;", body)
    assert len(re.findall(r"mbar_wait\(", body)) == 2
    assert re.search(r"if \(threadIdx.x == 0\) \{[^}]*mbar_wait\(empty\(prev\)", body)
