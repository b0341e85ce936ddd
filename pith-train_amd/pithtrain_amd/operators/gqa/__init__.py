"""The GQA layer while it answers: its key-value cache and attention to it (kv_cache.py)."""
