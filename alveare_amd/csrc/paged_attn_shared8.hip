// Attention of sequences that share their first pages: 8-bit pages.
#include "paged_attn_shared.h"

int alv::attention_shared8(const SharedCall& c) { return attention_shared<true>(c); }
