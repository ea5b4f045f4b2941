"""The language-model kernel templates compile for sm_100a with NVRTC, in every
variant that the operators can ask for by type, width and shape of a call."""
import ctypes
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SIZE = {"ga_half": 2, "ga_float": 4, "ga_double": 8}


def compiles(api, defines, template):
    text = '#include "cluda.h"\n' + "".join("#define %s %s\n" % d for d in defines) + '#include "%s"\n' % template
    size, log = ctypes.c_size_t(), ctypes.c_char_p()
    err = api.lib().gpuarray_b200_compile_check(text.encode(), None, os.path.join(ROOT, ".kernel_cache").encode(),
                                                ctypes.byref(size), ctypes.byref(log))
    assert err == 0 and size.value > 0, (log.value or b"").decode(errors="replace")[-3000:]


@pytest.mark.parametrize("build", ["GA_EM_BUILD_LOOKUP", "GA_EM_BUILD_GRAD"])
@pytest.mark.parametrize("a,o", [("ga_half", "ga_half"), ("ga_float", "ga_float"), ("ga_half", "ga_float"), ("ga_double", "ga_half"), ("ga_half", "ga_double")])
@pytest.mark.parametrize("accumulate", [0, 1])
def test_embedding(api, build, a, o, accumulate):
    widest = 16 // SIZE[a]
    while widest * SIZE[o] > 32:
        widest //= 2
    f = "ga_double" if "ga_double" in (a, o) else "ga_float"
    for e, rounds, cluster in ((widest, 2, 8), (1, 1, 1)):
        compiles(api, [(build, ""), ("GA_EM_A_T", a), ("GA_EM_O_T", o), ("GA_EM_I_T", "ga_ulong"), ("GA_EM_F_T", f), ("GA_EM_E", e),
                       ("GA_EM_C", max(1, 16 // (e * SIZE[a]))), ("GA_EM_ND", 4), ("GA_EM_ACCUMULATE", accumulate),
                       ("GA_EG_ROUNDS", rounds), ("GA_EG_CLUSTER", cluster)], "ga_embed.cuh")


@pytest.mark.parametrize("z", ["ga_half", "ga_float"])
@pytest.mark.parametrize("contig", [0, 1])
@pytest.mark.parametrize("top", [0, 1])
def test_log_probabilities(api, z, contig, top):
    common = [("GA_LP_Z_T", z), ("GA_LP_ZTYPE", int(z == "ga_float")), ("GA_LP_I_T", "ga_int"), ("GA_LP_ND", 2), ("GA_LP_CONTIG", contig)]
    for ent in (0, 1):
        for threads, group, cluster in ((128 if top else 256, 32, 1), (128, 128, 1), (256, 256, 2), (512, 512, 8)):
            compiles(api, [("GA_LP_BUILD_ROWS", "")] + common + [("GA_LP_ENT", ent), ("GA_LP_THREADS", threads), ("GA_LP_GROUP", group),
                     ("GA_LP_CLUSTER", cluster), ("GA_LP_TOP", top), ("GA_LP_FOLD", int(z == "ga_half" and not contig))], "ga_logprobs.cuh")
        if not top:
            for g in {z, "ga_float"}:
                compiles(api, [("GA_LP_BUILD_GRAD", "")] + common + [("GA_LP_ENT", ent), ("GA_LP_G_T", g), ("GA_LP_GTYPE", int(g == "ga_float"))],
                         "ga_logprobs.cuh")


@pytest.mark.parametrize("entries", [32, 128, 960])
def test_clipping(api, entries):
    compiles(api, [("GA_CN_CAP", entries)], "ga_clipnorm.cuh")
