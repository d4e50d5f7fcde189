"""A CTA of the adapter kernel whose wait for the other CTAs' sums runs out reports it and stays until their stores into its shared memory are in,
whatever its adapter's rank and whether it has rows in the second product.

Running such a case needs a kernel that fails, so the rule is checked on the source: from the wait on, its answer is only made one for the CTA, and the
first thing that is done with it is to report, to wait for the stores again, for this CTA's own copies too, to give tensor memory back and to leave."""
import importlib
import os
import re

import pytest

EXCHANGE = "ok = ptx::mbar_wait(bar, 0, abort_flag);"
MARKS = ["cp_async_wait<0>()", "atomicOr(&g_dense_err, ERR_WAIT_FOLD)", "*abort_flag = 0", "ptx::mbar_wait(bar, 0, abort_flag)", "__syncthreads()", "ptx::tmem_dealloc(", "return;"]


def _kernel(pkg):
    bld = importlib.import_module(pkg.__name__ + ".build")
    text = re.sub(r"//[^\n]*", "", open(os.path.join(bld.CSRC, "adapters.inl")).read())
    text = text[text.index("adapters_kernel(const __grid_constant__"):]
    return text[:text.index("\n}  // namespace") if "\n}  // namespace" in text else text.index("\nnamespace {")]


def _block(text, at):
    start = text.index("{", at)
    depth = 0
    for i in range(start, len(text)):
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        if depth == 0:
            return text[start:i + 1]
    raise ValueError("unbalanced braces")


def _misses(kernel):
    """What the way from the exchange's wait to its report lacks."""
    rest = kernel[kernel.index(EXCHANGE) + len(EXCHANGE):]
    at = re.search(r"\bif \(!ok\)", rest)
    ahead, bad = rest[:at.start()], []
    if re.findall(r"\bok = [^;]*;", ahead) != ["ok = __syncthreads_and(ok);"]:
        bad.append("the answer is combined with something")
    if re.search(r"\breturn\b|\bok\s*&&|&&\s*ok\b", ahead):
        bad.append("a way past the report")
    if rest[at.end():].lstrip()[0] != "{":
        return bad + ["no report"]
    report = _block(rest, at.end())
    where = [report.find(m) for m in MARKS]
    if -1 in where or where != sorted(where):
        bad.append("the report is not " + ", ".join(MARKS))
    if "rank" in report or "first" in report or "end" in report:
        bad.append("the report depends on rank or rows")
    return bad


def test_a_wait_for_sums_that_runs_out_is_reported_whatever_rank_and_rows(pkg):
    assert _misses(_kernel(pkg)) == []


def test_the_products_are_waited_for_before_tensor_memory_is_given_back(pkg):
    kernel = _kernel(pkg)
    rest = kernel[kernel.index(EXCHANGE):]
    tail = rest[rest.index("ok = __syncthreads_and(ok);", rest.index("add_to4(")):]
    report = _block(tail, tail.index("if (tid == 0 && !ok)"))
    assert "atomicOr(&g_dense_err, ERR_WAIT_FOLD)" in report and re.search(r"for \(int k = max\(0, issued - 2\); k < issued; \+\+k\)", report)
    assert report.index("*abort_flag = 0") < report.index("ptx::mbar_wait(bar + 8 + 8 * (k & 1), (k >> 1) & 1, abort_flag)")
    assert tail.index("if (tid == 0 && !ok)") < tail.index("__syncthreads();") < tail.index("ptx::tmem_dealloc(tmem, 256)")


def test_the_check_itself():
    good = EXCHANGE + " f(); ok = __syncthreads_and(ok); if (!ok) { " + "; ".join(MARKS) + " }"
    assert _misses(good) == []
    assert _misses(good.replace("ok = __syncthreads_and(ok);", "ok = __syncthreads_and(ok && wanted);"))
    assert _misses(good.replace("f();", "ok = __syncthreads_and(ok && wanted);"))
    assert _misses(good.replace("f();", "if (rank == 0) return;"))
    assert _misses(good.replace("ptx::mbar_wait(bar, 0, abort_flag); __", "__"))
    assert _misses(good.replace("*abort_flag = 0", "if (first < rows) *abort_flag = 0"))


@pytest.mark.gpu
def test_the_report_names_the_adapters(pkg):
    """They share the projection's word, so its text must not send the reader to the projection alone. (The codes come from the wait self-test.)"""
    torch = pytest.importorskip("torch")
    api = importlib.import_module(pkg.__name__ + ".api")
    assert api.dense_status() == 0
    waited = torch.zeros(6, dtype=torch.int64, device="cuda")
    api._check(api.lib().llattn_wait_selftest(1_000_000, api.dense_error_word(), waited.data_ptr(), None))
    torch.cuda.synchronize()
    with pytest.raises(api.LlattnError, match="projection or of its adapters"):
        api.dense_status()
    assert api.dense_status() == 0
