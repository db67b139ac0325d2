# SPDX-License-Identifier: MIT
"""beamgrad_amd: differentiable beam search on AMD Instinct MI355X (gfx950).

A drop-in for beamgrad's GPU path: the same Python API (``decode``,
``final_scores``, ``backtrack``, ``search``, ``beam_search``,
``length_penalty``, ``losses``) and the same ``torch.ops.beamgrad`` operators,
served by hand-written HIP kernels in ``libdbs_hip`` (whose C ABI is the
reference's ``dbs_cuda.h``). Beside them, the state of the model that is
searched: attention over a paged cache (``tree_attention``), the cache's pages
(``PageTable``, ``fork_pages``, ``extend_pages``, ``write_tokens``,
``keep_tokens``), its eviction by the attention that tokens got
(``accumulate_weights``, ``evict_tokens``), rotary positions (``rotary``), dense states
in the order of the beams (``reorder_states``), and the log-probabilities of given
tokens (``token_logprobs``).

The public names load on first use. Importing the package itself loads
nothing, so ``beamgrad_amd._C_hip`` (the operators' HIP kernels) can be
imported on its own beside another package that owns the operators and
their Python registrations (the reference's ``_C`` and ``_torch.py``).
"""

from __future__ import annotations

import importlib

__version__ = "0.1.0"

# public name -> the module that defines it
_PUBLIC = {
    "BeamOptions": "._options",
    "CUDA_MAX_BEAM": "._options",
    "BeamSearchResult": "._search",
    "BeamState": "._search",
    "beam_search": "._search",
    "search": "._search",
    "sequence_scores": "._search",
    "TokenLogprobs": "._scores",
    "token_logprobs": "._scores",
    "PageTable": "._cache",
    "accumulate_weights": "._cache",
    "evict_tokens": "._cache",
    "extend_pages": "._cache",
    "fork_pages": "._cache",
    "keep_tokens": "._cache",
    "reorder_states": "._cache",
    "rotary": "._cache",
    "rotary_frequencies": "._cache",
    "tree_attention": "._cache",
    "write_tokens": "._cache",
    "BeamSearchOutput": "._torch",
    "backtrack": "._torch",
    "cuda_available": "._torch",
    "decode": "._torch",
    "final_scores": "._torch",
    "length_penalty": "._torch",
}

__all__ = sorted([*_PUBLIC, "losses", "__version__"])


def __getattr__(name: str):
    if name == "losses":
        value = importlib.import_module(".losses", __name__)
    elif name in _PUBLIC:
        value = getattr(importlib.import_module(_PUBLIC[name], __name__), name)
    else:
        raise AttributeError(f"module {__name__!r} has no attribute {name!r}")
    globals()[name] = value
    return value


def __dir__():
    return sorted(set(globals()) | set(__all__))
