// kvb_pages_host.h - what the host code of the paged cache's translation units shares.
#pragma once

#include "kvb_host.h"
#include "kvb_pages_view.cuh"

namespace kvbh {

// KVB_OK, or what is wrong with a pool's descriptor (message names the entry point `who`).
kvb_status check_pages(const char* who, const kvb_pages* p);
kvb::PagesView view_of(const kvb_pages* p);

}  // namespace kvbh
