"""Model registry: a model folder's config.json names its architecture; the registry maps it to the loader."""
from __future__ import annotations

import json
from pathlib import Path

from . import galirax, genesun, mafuzen, medodra, tugezen, zevopel
from .lib import B200Error

ARCHITECTURES = {
    "Genesun": genesun.load,
    "Galirax": galirax.load,
    "Zevopel": zevopel.load,
    "Medodra": medodra.load,
    "Mafuzen": mafuzen.load,
    "Tugezen": tugezen.load,
}


PAGED = ("Galirax",)  # architectures whose caches may be kept in 8 bits, in pages (kv8_page)


def load_model(path, **kw):
    """Load the model in `path` with the loader of its architecture (kw: dtype, n_ctx, n_seq_max, max_batch, device; kv8_page for those in PAGED)."""
    cfg = json.loads((Path(path) / "config.json").read_text())
    arch = cfg.get("architecture")
    if arch not in ARCHITECTURES:
        raise B200Error(f"{path}: architecture {arch!r} is not one of {sorted(ARCHITECTURES)}")
    if arch not in PAGED and kw.pop("kv8_page", 0):
        raise B200Error(f"{path}: architecture {arch} keeps no 8-bit pages (kv8_page): {', '.join(PAGED)} only")
    return ARCHITECTURES[arch](path, **kw)
