"""The build looks at what registers the compiler gave to kernels whose warps hand registers to one another."""
import pytest

from xcalibur_b200 import build


def report(kernels):
    return "".join(f"ptxas info    : Compiling entry function '{name}' for 'sm_100a'\n"
                   f"ptxas info    : Function properties for {name}\n"
                   f"    0 bytes stack frame, 0 bytes spill stores, 0 bytes spill loads\n"
                   f"ptxas info    : Used {regs} registers, used 2 barriers\n" for name, regs in kernels)


def names(f8=1, dims=(64, 128), rows=(1, 2)):
    return [f"_ZN3xcb11attn_kernelI{t}Lb{f8}ELi{d}ELi{w}EEEvNS_10AttnParamsE" for t in ("6__half", "13__nv_bfloat16")
            for d in dims for w in rows]


def test_register_split():
    others = [(n, 168) for n in names(f8=0) + names(dims=(256,)) + names(rows=(4, 8))]
    good = [(n, 128) for n in names()]
    build.check_register_split(report(others + good))
    build.check_register_split(report(good[:3] + [(good[3][0], 121)] + others + good[4:]))  # given out by eights
    for bad in (good[:-1], good[:-1] + [(good[-1][0], 120)], good[:-1] + [(good[-1][0], 136)], []):
        with pytest.raises(RuntimeError):
            build.check_register_split(report(others + bad))
