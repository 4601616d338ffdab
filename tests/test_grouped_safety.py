"""CPU: rules of the grouped kernel whose breach could hang the GPU or race on
its memory, checked on the source and on the plans.  No GPU is touched."""

from __future__ import annotations

import re
import subprocess

import pytest

from test_kernel_layout import CSRC, ROOT, _nvcc


def _code(name):
    """A source file without its comments."""
    text = (CSRC / name).read_text()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    return re.sub(r"//[^\n]*", "", text)


def _kernel():
    code = _code("tinym_grouped.cuh")
    return code[code.index("tinym_grouped_kernel("):]


def test_tensor_memory_is_allocated_between_wait_and_trigger():
    """No CTA holds tensor memory while it waits for the grid before, and no
    dependent CTA can come to an SM before this grid's CTA there has its own:
    else each could hold what the other waits for."""
    kernel = _kernel()
    wait, alloc, trigger = (kernel.index(s) for s in
                            ("grid_dependency_wait()", "Ops::alloc(", "grid_launch_dependents()"))
    assert wait < alloc < trigger
    assert kernel.count("Ops::alloc(") == kernel.count("grid_launch_dependents()") == 1
    # by the allocating warp alone: `if (warp == 1) { alloc; trigger }`
    between = kernel[kernel.rindex("if (warp == 1) {", 0, alloc):trigger]
    assert "}" not in between


def test_plans(tmp_path):
    nvcc = _nvcc()
    if nvcc is None:
        pytest.skip("nvcc not found")
    exe = tmp_path / "grouped_safety_host"
    build = subprocess.run(
        [nvcc, "-std=c++17", "-O1", "-gencode", "arch=compute_100a,code=sm_100a", "-I", str(CSRC),
         "-I", str(ROOT / "include"), str(ROOT / "tests" / "grouped_safety_host.cu"), "-o", str(exe)],
        capture_output=True, text=True, timeout=600)
    assert build.returncode == 0, build.stderr[-4000:]
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stdout[-4000:]
    assert run.stdout.startswith("grouped safety checks ok ("), run.stdout


def test_other_ctas_barriers_are_signalled_at_cluster_scope():
    """What one CTA of a pair wrote is ordered before the other's use of it:
    a thread that arrives on the other CTA's barrier releases at cluster scope
    (the arrival itself, or a fence in front of it), and a wait on a barrier
    that the other CTA signals acquires at it.  Copies and MMAs signal by
    themselves, at cluster scope by definition."""
    code = _code("tinym_grouped.cuh")
    # one spelling of an arrival on another CTA's barrier
    assert len(re.findall(r"mbarrier\.arrive[\w.:]*shared::cluster", code)) == 1
    body = code[code.index("void mbar_arrive_remote("):]
    body = body[:body.index("}")]
    arrive = re.search(r"mbarrier\.arrive\.(\w+)\.cluster\.shared::cluster", body)
    assert arrive
    if arrive.group(1) == "relaxed":
        fence = re.search(r"fence\.(acq_rel|release)[\w.:]*\.cluster;", body)
        assert fence and fence.start() < arrive.start()
    else:
        assert arrive.group(1) == "release"
    assert "mbarrier.try_wait.parity.acquire.cluster" in code
    kernel = _kernel()
    # threads announce their own stores (scales) and what they have read
    # (accumulators); they pass nothing on
    announced = re.findall(r"mbar_arrive_remote\(at_rank\((\w+)", kernel)
    assert sorted(announced) == ["acc_empty", "full_bar"]
    # every wait acquires at cluster scope in a pair kernel; the one without is
    # in the scale warps of the others
    scopes = re.findall(r"warp_wait(<\w+>)?\(", kernel)
    assert scopes.count("") == 1 and set(scopes) == {"", "<PAIR>", "<true>"}
    assert "warp_wait(empty_bar(s)" in kernel[kernel.index("if constexpr (FP4 && !PAIR)"):]


def test_teardown_decides_on_draining_when_every_role_has_ended():
    """A wait of any role may run out after the producer or the MMA warp has
    finished: whether copies and MMAs in flight are waited for is decided
    behind the barrier at which the roles meet, before tensor memory is freed."""
    kernel = _kernel()
    meet = kernel.index("meet();")
    drains = [m.start() for m in re.finditer(r"mbar_drain\(", kernel)]
    assert len(drains) >= 2 and all(meet < d < kernel.index("Ops::dealloc(") for d in drains)
    assert kernel.count("*abort_flag != 0") == 1 and kernel.index("*abort_flag != 0") > meet


def test_selftest_refusals():
    import tinym_b200

    lib, p = tinym_b200.capi(), 1 << 20
    for lost, xs, ws, ns in [(3, None, None, 1000), (-1, p, p, 1000), (0, p, None, 1000),
                             (1, None, p, 1000), (2, p, p, 0), (2, p, p, 10 ** 11)]:
        assert lib.tinym_selftest_grouped_lost(lost, p, xs, p, ws, p, 4, 2, 64, 64, p, ns, None) == 1


def test_kernels_that_start_early_use_no_read_only_loads():
    """A kernel launched while the one before still writes its inputs may not
    read them as memory that stays as it is for the kernel's whole run (.nc,
    __ldg), not even behind the dependency wait."""
    for name in ("tinym_grouped.cuh", "tinym_mxfp4.cuh", "tinym_kernels.cuh"):
        code = _code(name)
        if name == "tinym_kernels.cuh":  # launched after the kernel before has ended
            code = code[:code.index("tinym_pack_weights_kernel")]
        assert "global.nc" not in code and "__ldg" not in code, name
