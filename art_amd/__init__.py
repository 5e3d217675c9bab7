"""art_amd: MI355X-native exact MIPS top-k search behind ART's evidence-index API.

Public surface (mirrors /root/reference/megatron/data/art_index.py):
    detach, OpenRetreivalDataStore, DistributedBruteForceIndex
Engine level (ctypes over include/artmips.h):
    art_amd.engine.MipsEngine, art_amd.distributed.spmd_search
What reads the passages a search found (ctypes over include/arttok.h and include/artread.h):
    art_amd.token_store.DeviceTokenStore, art_amd.reader.embed_tokens, art_amd.reader.cross_attention
"""
from .art_index import DistributedBruteForceIndex, OpenRetreivalDataStore, detach

__all__ = ["detach", "OpenRetreivalDataStore", "DistributedBruteForceIndex"]
__version__ = "0.1.0"
