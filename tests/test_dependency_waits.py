"""Kernels that are launched before the one in front of them has ended (programmatic dependent launch) store nothing to global memory until they
have waited for it: what lies there may still be read, or written, by that kernel.  The allocator hands memory on in stream order, so that the scratch of a call
can be what the kernel in front still works on."""

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "mlx_turboquant_b200" / "csrc"
# The expansion of a prefill stores from its start: it only ever follows the query kernel of the same call, which lets it start behind its own wait and touches none of
# what the expansion writes (checked below).  A job that `follows` another one of the same call waits at its end: the jobs' results are their own.
FOLLOWERS = {"fa_expand_kernel", "dequantize_tc_kernel", "quantize_tc_kernel"}
WAIT = re.compile(r"\bpdl_wait\(\)|griddepcontrol\.wait")


def kernels():
    for path in sorted([*CSRC.glob("*.cu"), *CSRC.glob("*.cuh")]):
        code = re.sub(r"//[^\n]*", "", path.read_text())
        for m in re.finditer(r"__global__\s+void\s+(?:__launch_bounds__\((?:[^()]|\([^()]*\))*\)\s*)?(\w+)\s*\(", code):
            end = code.find("\n}", m.end())
            yield path.name, m.group(1), code[m.end():end]


WAITING = [(file, name, body) for file, name, body in kernels() if WAIT.search(body)]


def stores_before(prefix: str) -> list[str]:
    """Stores through pointers, in code that runs before a wait, to anything but shared memory and the thread's own arrays."""
    own = set(re.findall(r"\b[A-Za-z_]\w*[*&]?[ ]+(\w+)(?:\[[^\]=;]*\])+\s*[=;,{]", re.sub(r"\b(return|else)\b", ";", prefix)))      # arrays, declared here
    own |= set(re.findall(r"\]\s*,\s*(\w+)\[[^\]=;]*\]\s*[,;]", prefix))                                           # ... further ones of a list
    own |= set(re.findall(r"\b(\w+)\s*=\s*[^;]*\b(?:smem\w*|gp|fp|tab|s_misc|qs|qf|us|ctab|rs)\b[^;]*;", prefix))     # pointers into shared memory
    own |= set(re.findall(r"\b(\w+) = reinterpret_cast<\w+\*>\(t\w* ", prefix))
    found = []
    for m in re.finditer(r"\*\s*reinterpret_cast<[^<>]*\*>\(\s*([^;]*?)\)\s*=(?!=)|(?:^|[;{}\s(])(\w+)\[[^;{}]*?\]\s*[-+|]?=(?!=)|\b(atomic\w+|store\w*|__st\w+)\s*(?:<\w+>)?\(|\"(st\.global|red\.|atom\.)", prefix):
        target = re.match(r"\w+", (m.group(1) or m.group(2) or "").strip())
        if (m.group(1) or m.group(2)) and target and (target.group() in own or target.group() in ("smem", "slot")):
            continue
        found.append(m.group().strip())
    return found


def test_the_kernels_are_found():
    assert {"blocks_fa_expand_kernel", "blocks_fa_kernel", "blocks_write_kernel", "rotary_kernel", "decode_lane_kernel", "fa_query_kernel"} <= {name for _, name, _ in WAITING}


def test_a_store_before_the_wait_is_seen():
    assert stores_before("float* scales = p.scales + at; if (tid == 0) *reinterpret_cast<int2*>(scales + 2) = make_int2(1, 2);")
    assert stores_before("float* part = p.part; part[tid] = 0.f;") and stores_before("atomicAdd(p.count, 1);") and stores_before("store_from_f32(p.out, 0, 1, 2.f);")
    assert not stores_before("float x[4]; x[0] = 1.f; unsigned char* s = smem + 4; *reinterpret_cast<int*>(s + 8) = 1; slot[1] = 0u;")


@pytest.mark.parametrize("file,name,body", [pytest.param(*k, id=k[1]) for k in WAITING if k[1] not in FOLLOWERS])
def test_no_store_before_the_wait(file, name, body):
    prefix = body[:WAIT.search(body).start()]
    # a plan that the host has already refused: the status word alone, and the kernel ends
    prefix = re.sub(r"atomicCAS\((?:&g_status|p\.status), 0, ERR_LAYOUT\);\s*return;", "", prefix)
    assert stores_before(prefix) == [], f"{file}: {name}"


def test_the_expansion_of_a_prefill_follows_a_kernel_that_has_waited():
    text = (CSRC / "prefill_fa.cu").read_text()
    body = next(b for f, n, b in WAITING if n == "fa_query_kernel")
    assert body.index("pdl_wait()") < body.index("pdl_trigger()")
    assert text.index("? fa_query_kernel<D, NC_FEW> : fa_query_kernel<D, NC>") < text.index("cudaLaunchKernelEx(&cfg, fa_expand_kernel<D>, e)")
