from .manager import (CacheError, CacheFull, KVRequirement, StateRequirement, PagePool, KVGroup,
                      CacheManager)
from .kv8 import Kv8Cache, Kv8Plan
