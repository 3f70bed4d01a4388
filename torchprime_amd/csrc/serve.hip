// The operators that answer with a model: the paged key-value cache, attention over it, sampling.
#include "kv_cache.hpp"
#include "paged_attn.hpp"
#include "sample.hpp"
